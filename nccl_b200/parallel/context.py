"""Context (sequence) parallelism recipes over the library's point-to-point and all-to-all calls.

ring_attention   every rank holds a contiguous slice of the sequence. Key / value blocks travel
                 round the ring with one grouped ncclSend + ncclRecv per step into a second buffer
                 while the current block is being used (double buffering; on a GPU the exchange runs
                 on a communication stream). Partial results are merged with the running-maximum
                 ("online softmax") update, so the result equals attention over the whole sequence.
ulysses_*        all-to-all that swaps the sharded dimension: from "sequence sharded, all heads"
                 to "all of the sequence, heads sharded" before attention and back after it.

The attention arithmetic is plain PyTorch unless a ``ContextParallel`` (nccl_b200.ops.cp) is given as ``cp``: then it is that one's kernels (fp16 or bf16 on the
communicator's GPU), which never hold a block's scores in memory. Either way there is a backward pass, written out as the forward is:

    out, lse = ring_attention(comm, q, k, v, causal=True, cp=cp, with_lse=True)
    dq, dk, dv = ring_attention_backward(comm, dout, q, k, v, out, lse, causal=True, cp=cp)
    out, state = ulysses_attention(comm, q, k, v, causal=True, cp=cp, with_state=True)
    dq, dk, dv = ulysses_attention_backward(comm, dout, state, causal=True, cp=cp)

With ``cp`` results have no history for autograd, also where inputs require gradients: those come from the backward calls. (Without it they have the local one, which knows
nothing of what other ranks do with this rank's keys and values.)

Reference parity: the reference ships the primitives only (grouped ncclSend / ncclRecv ring of docs/examples/02_point_to_point/01_ring_pattern,
ncclAlltoAll of src/collectives.cc).
"""
import math

import torch

from ..core import group


def _block(q, k, v, scale, mask):
    """Scores of one key / value block: returns (block maximum, exp-sum, unnormalised output), fp32."""
    s = torch.matmul(q.float(), k.float().transpose(-1, -2)) * scale          # [B, H, Sq, Sk]
    if mask is not None:
        s = s.masked_fill(~mask, float("-inf"))
    m = s.amax(dim=-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)                    # fully masked rows
    p = torch.exp(s - m)
    if mask is not None:
        p = p.masked_fill(~mask, 0.0)
    return m, p.sum(dim=-1, keepdim=True), torch.matmul(p, v.float())


def _block_backward(q, k, v, dout, lse, delta, scale, mask):
    """What one key / value block adds to (dq, dk, dv), fp32; the probabilities come from the scores and the log-sum-exp over all keys."""
    p = torch.exp(torch.matmul(q.float(), k.float().transpose(-1, -2)) * scale - lse[..., None])
    if mask is not None:
        p = p.masked_fill(~mask, 0.0)
    ds = p * (torch.matmul(dout.float(), v.float().transpose(-1, -2)) - delta[..., None]) * scale
    return torch.matmul(ds, k.float()), torch.matmul(ds.transpose(-1, -2), q.float()), torch.matmul(p.transpose(-1, -2), dout.float())


def _rows(t):
    """[batch, heads, sequence, dim] as the kernels take it, [batch, sequence, heads, dim]; a copy where its rows are not where they can be read."""
    t = t.transpose(1, 2)
    fits = t.stride(3) == 1 and t.data_ptr() % 16 == 0 and all(n == 1 or (s > 0 and s % 8 == 0) for n, s in zip(t.shape, t.stride()[:3]))
    return t if fits else t.clone(memory_format=torch.contiguous_format)   # (a contiguous tensor may be off the grid)


class _Ring:
    """Passes a tensor on to the next rank and takes the previous one's into another, on a GPU on a stream of its own. `device`: the tensors', which need not be the current one."""

    def __init__(self, comm, cuda, device, stream):
        self.comm, self.cuda, self.device = comm, cuda, device
        self.nxt, self.prv = (comm.rank + 1) % comm.nranks, (comm.rank - 1) % comm.nranks
        self.stream = stream if stream is not None else (torch.cuda.Stream(device=device) if cuda and comm.nranks > 1 else None)

    def pass_on(self, send, recv):
        """Behind what the device's current stream has been given so far; gives what to wait for before `recv` is read or `send` written (None: it is done)."""
        comm = self.comm
        if not self.cuda:
            with group(comm.lib):
                comm.send(send, self.nxt)
                comm.recv(recv, self.prv)
            return None
        ready = torch.cuda.Event()
        ready.record(torch.cuda.current_stream(self.device))   # `recv` is no longer read, `send` is complete
        with torch.cuda.stream(self.stream):
            self.stream.wait_event(ready)
            with group(comm.lib):
                comm.send(send, self.nxt, stream=self.stream)
                comm.recv(recv, self.prv, stream=self.stream)
            done = torch.cuda.Event()
            done.record(self.stream)
        return done

    def wait(self, done):
        if done is not None:
            torch.cuda.current_stream(self.device).wait_event(done)


def ring_attention(comm, q, k, v, causal=False, stream=None, cp=None, with_lse=False):
    """q, k, v: [batch, heads, local sequence, head dim]; rank r holds positions [r * S, (r + 1) * S).
    Returns this rank's slice of softmax(q k^T / sqrt(d)) v over the whole sequence, in q's dtype; ``with_lse`` also the fp32 log-sum-exp
    [batch, heads, local sequence] that ``ring_attention_backward`` takes. With ``cp`` k and v may have fewer heads, which groups of q's share."""
    n, rank = comm.nranks, comm.rank
    scale = 1.0 / math.sqrt(q.shape[-1])
    S = q.shape[2]
    kv = [torch.stack((k, v)).contiguous(), None]
    kv[1] = torch.empty_like(kv[0])
    ring = _Ring(comm, q.is_cuda, q.device, stream)
    if cp is None:
        m_run = torch.full(q.shape[:3] + (1,), float("-inf"), dtype=torch.float32, device=q.device)
        l_run = torch.zeros_like(m_run)
        o_run = torch.zeros(q.shape, dtype=torch.float32, device=q.device)
        tri = torch.ones(S, S, dtype=torch.bool, device=q.device).tril() if causal else None
    else:
        rows, joined = _rows(q), None
        last = rank if causal else n - 1            # the last step that has something to add here
    for step in range(n):
        cur, other = kv[step % 2], kv[(step + 1) % 2]
        done = ring.pass_on(cur, other) if step + 1 < n else None   # the block goes on while it is being used here
        src = (rank - step) % n                     # the rank whose keys / values are in `cur`
        if causal and src > rank:
            pass
        elif cp is not None:
            own = causal and src == rank
            joined = cp.attention(rows, cur[0].transpose(1, 2), cur[1].transpose(1, 2), causal=own, offset=0 if own else None, join=joined,
                                  dtype=q.dtype if step == last else torch.float32)
        else:
            mask = tri if causal and src == rank else None
            m_blk, l_blk, o_blk = _block(q, cur[0], cur[1], scale, mask)
            m_new = torch.maximum(m_run, m_blk)
            a_old = torch.exp(m_run - m_new)
            a_blk = torch.exp(m_blk - m_new)
            l_run = l_run * a_old + l_blk * a_blk
            o_run = o_run * a_old + o_blk * a_blk
            m_run = m_new
        ring.wait(done)
    if cp is not None:
        out, lse = joined[0].transpose(1, 2), joined[1]
        return (out, lse) if with_lse else out
    out = (o_run / l_run).to(q.dtype)
    return (out, (m_run + torch.log(l_run))[..., 0]) if with_lse else out


def ring_attention_backward(comm, dout, q, k, v, out, lse, causal=False, stream=None, cp=None):
    """(dq, dk, dv) of ``ring_attention`` for this rank's slices, in q's dtype, from the gradient of its result; out and lse as it returned them.
    The blocks go round as before, and with each go the gradients that the ranks so far have added for it, in fp32: behind the last step they
    are back at the rank that the block belongs to."""
    n, rank = comm.nranks, comm.rank
    scale = 1.0 / math.sqrt(q.shape[-1])
    S = q.shape[2]
    kv = [torch.stack((k, v)).contiguous(), None]
    kv[1] = torch.empty_like(kv[0])
    ring = _Ring(comm, q.is_cuda, q.device, stream)
    # gradients of the block that is here, and where the next one's arrive; with kernels [.., sequence, heads, dim]
    shape = kv[0].shape if cp is None else kv[0].transpose(2, 3).shape
    grads = [torch.empty(shape, dtype=torch.float32, device=q.device) for _ in range(2)]
    if cp is None:
        delta = (dout.float() * out.float()).sum(-1)
        tri = torch.ones(S, S, dtype=torch.bool, device=q.device).tril() if causal else None
        dq = torch.zeros(q.shape, dtype=torch.float32, device=q.device)
    else:
        rows, drows = _rows(q), _rows(dout)
        delta, dq = cp.attention_delta(drows, _rows(out)), torch.empty(rows.shape, dtype=torch.float32, device=q.device)
        lse = lse.contiguous()
    grads_done = None
    for step in range(n):
        cur, other = kv[step % 2], kv[(step + 1) % 2]
        g = grads[step % 2]
        done = ring.pass_on(cur, other) if step + 1 < n else None
        src = (rank - step) % n
        ring.wait(grads_done)
        if causal and src > rank:
            pass                                    # nothing of this block is visible here: its gradients only pass through
        elif cp is not None:
            own = causal and src == rank
            cp.attention_backward(drows, rows, cur[0].transpose(1, 2), cur[1].transpose(1, 2), None, lse, causal=own, offset=0 if own else None, delta=delta,
                                  add=(dq, g[0], g[1]) if step else None, dtype=torch.float32, dq=dq, dk=g[0], dv=g[1])
        else:
            add = _block_backward(q, cur[0], cur[1], dout, lse, delta, scale, tri if causal and src == rank else None)
            dq += add[0]
            if step:
                g[0] += add[1]
                g[1] += add[2]
            else:
                g[0].copy_(add[1])
                g[1].copy_(add[2])
        if n > 1:
            grads_done = ring.pass_on(g, grads[(step + 1) % 2])
        ring.wait(done)
    ring.wait(grads_done)
    g = grads[n % 2 if n > 1 else 0].to(q.dtype)
    dq = dq.to(q.dtype)
    return (dq, g[0], g[1]) if cp is None else (dq.transpose(1, 2), g[0].transpose(1, 2), g[1].transpose(1, 2))


def ulysses_scatter_heads(comm, x, stream=None):
    """[batch, local sequence, heads, dim] on every rank -> [batch, sequence, heads / n, dim]:
    rank r ends up with heads [r * H / n, (r + 1) * H / n) of every position. One ncclAlltoAll."""
    n = comm.nranks
    B, S, H, D = x.shape
    if H % n:
        raise ValueError("the number of heads must be a multiple of the number of ranks")
    if n == 1:
        return x
    send = x.reshape(B, S, n, H // n, D).permute(2, 0, 1, 3, 4).contiguous()    # [n, B, S, H/n, D]: block p goes to rank p
    recv = torch.empty_like(send)
    comm.all_to_all(send, recv, stream=stream)                                   # block p now holds rank p's positions
    return recv.permute(1, 0, 2, 3, 4).reshape(B, n * S, H // n, D)


def ulysses_gather_heads(comm, x, stream=None):
    """Inverse of ulysses_scatter_heads: [batch, sequence, heads / n, dim] -> [batch, local sequence, heads, dim]."""
    n = comm.nranks
    B, S_all, Hl, D = x.shape
    if S_all % n:
        raise ValueError("the sequence length must be a multiple of the number of ranks")
    if n == 1:
        return x
    S = S_all // n
    send = x.reshape(B, n, S, Hl, D).permute(1, 0, 2, 3, 4).contiguous()         # [n, B, S, H/n, D]: block p = rank p's positions
    recv = torch.empty_like(send)
    comm.all_to_all(send, recv, stream=stream)                                   # block p now holds rank p's heads
    return recv.permute(1, 2, 0, 3, 4).reshape(B, S, n * Hl, D)


def _whole_sequence(q, k, v, causal):
    """Probabilities of [batch, heads, sequence, dim] in fp32."""
    s = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(q.shape[-1])
    if causal:
        s = s.masked_fill(~torch.ones(s.shape[-2:], dtype=torch.bool, device=s.device).tril(), float("-inf"))
    return torch.softmax(s, -1)


def ulysses_attention(comm, q, k, v, causal=False, cp=None, with_state=False):
    """q, k, v: [batch, local sequence, heads, dim]. Swaps to head sharding, runs full-sequence attention on
    this rank's heads, swaps back. Returns [batch, local sequence, heads, dim]; ``with_state`` also what ``ulysses_attention_backward`` takes. With ``cp`` k and v may
    have fewer heads (a multiple of the number of ranks)."""
    whole = [ulysses_scatter_heads(comm, t) for t in (q, k, v)]                           # [B, S_all, H/n, D]
    if cp is not None:
        whole = [_rows(t.transpose(1, 2)) for t in whole]                                 # (of one rank: as they were given)
        o, lse = cp.attention(*whole, causal=causal, offset=0 if causal else None)
    else:
        qh, kh, vh = (t.transpose(1, 2) for t in whole)
        o = torch.nn.functional.scaled_dot_product_attention(qh.float(), kh.float(), vh.float(), is_causal=causal).to(q.dtype).transpose(1, 2).contiguous()
        lse = None
    out = ulysses_gather_heads(comm, o)
    return (out, (*whole, o, lse)) if with_state else out


def ulysses_attention_backward(comm, dout, state, causal=False, cp=None):
    """(dq, dk, dv) of ``ulysses_attention``, [batch, local sequence, heads, dim] like its inputs, from the gradient of its result and what it kept."""
    qh, kh, vh, o, lse = state
    do = ulysses_scatter_heads(comm, dout)
    if cp is not None:
        grads = cp.attention_backward(_rows(do.transpose(1, 2)), qh, kh, vh, o, lse, causal=causal, offset=0 if causal else None)
    else:
        f = [t.float().transpose(1, 2) for t in (qh, kh, vh, do)]
        p = _whole_sequence(*f[:3], causal)
        dp = torch.matmul(f[3], f[2].transpose(-1, -2))
        ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(qh.shape[-1])
        grads = (torch.matmul(ds, f[1]), torch.matmul(ds.transpose(-1, -2), f[0]), torch.matmul(p.transpose(-1, -2), f[3]))
        grads = [t.to(qh.dtype).transpose(1, 2).contiguous() for t in grads]
    return tuple(ulysses_gather_heads(comm, t) for t in grads)
