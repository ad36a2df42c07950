"""GPU: the long-history operators where one part of a kernel meets another -- sinks beyond the window's reach, workgroups
of every size, the accuracy that bf16 is meant to have -- and calls at the edge of what is allowed.  The 64-bit forms, the
inputs and the counting of roundings are those of test_gpu_history_ops.py."""
import math

import pytest
import torch

from test_gpu_history_ops import check_window, rand

pytestmark = pytest.mark.gpu


def window_call(asme, dtype, b, n, h, kv, d, window, sinks, causal, valid, scale=None, seed=2):
    """inputs with junk in padding, (out, dq, dk, dv)"""
    q, k, v, dout = (rand(b, n, x, d, seed=seed + i, dtype=dtype, scale=1.5) for i, x in enumerate((h, kv, kv, h)))
    if valid is not None:
        for t, junk in ((q, math.nan), (k, math.inf), (v, math.nan), (dout, -math.inf)):
            t[~valid.cuda()] = junk
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    out = asme.ops.window_attention(q, k, v, window, sinks=sinks, causal=causal, scale=scale,
                                    valid=None if valid is None else valid.cuda())
    return (q, k, v, dout), [out, *torch.autograd.grad(out, (q, k, v), dout)]


def ragged(b, n, seed):
    """right padding of every length, a hole, and (of several) a sequence with nothing in it"""
    valid = torch.arange(n) < torch.randint(1, n + 1, (b, 1), generator=torch.Generator().manual_seed(seed))
    valid[:, n // 3] = False
    if b > 1:
        valid[1] = False
    return valid


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,n,h,kv,d,window,sinks,causal,padding", [
    # both directions: a query sees the sinks ahead of it too, however far beyond its window they lie -- workgroups of 64
    # queries, of 128 and of 256, sinks that end in the middle of a tile, and all positions sinks
    (2, 300, 2, 1, 64, 4, 200, False, True), (1, 500, 4, 2, 128, 4, 400, False, False),
    (2, 300, 2, 2, 32, 1, 129, False, False), (1, 1000, 2, 2, 16, 4, 200, False, True),
    (1, 400, 2, 1, 64, 3, 1000, False, True), (30, 300, 4, 2, 32, 5, 290, False, True),
    (11, 700, 4, 2, 64, 7, 600, False, True),
    # the same with many sinks behind the window's reach: tiles on both sides of theirs left to the far pass
    (1, 1200, 2, 1, 64, 5, 300, False, True), (1, 1200, 2, 1, 64, 5, 300, True, True)])
def test_window_attention_with_many_sinks(asme, dev, dtype, b, n, h, kv, d, window, sinks, causal, padding):
    valid = ragged(b, n, 1) if padding else torch.ones(b, n, dtype=torch.bool)
    (q, k, v, dout), got = window_call(asme, dtype, b, n, h, kv, d, window, sinks, causal, valid if padding else None)
    check_window(got, dtype, q, k, v, dout, window, sinks, causal, valid, d ** -0.5, n)
