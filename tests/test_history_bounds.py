"""CPU: the bounds that the GPU tests hold bf16 window attention to notice the mistakes that they are there for, planted in a
64-bit form of it."""
import math

import pytest
import torch

from test_gpu_history_edges import FEW_KEYS, check_close
from test_gpu_history_ops import rand, seen64


def rounded(t):
    return t.to(torch.bfloat16).double()


def same(t):
    return t


def attention(q, k, v, dout, window, sinks, causal, of_p=same, of_ds=same, of_out=same):
    """(out, dq, dk, dv), of_*: what becomes of P and dS as factors and of the output that D is formed from"""
    n, d, group = q.shape[1], q.shape[3], q.shape[2] // k.shape[2]
    q, k, v, dout = (t.double().transpose(1, 2) for t in (q, k, v, dout))
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    m = seen64(n, window, sinks, causal, torch.ones(q.shape[0], n, dtype=torch.bool))[:, None]
    p = torch.softmax((q @ k.transpose(-1, -2) * d ** -0.5).masked_fill(~m, -math.inf), -1)
    out = of_p(p) @ v
    ds = of_ds(p * (dout @ v.transpose(-1, -2) - (dout * of_out(out)).sum(-1, keepdim=True)))
    share = lambda t: t.unflatten(1, (-1, group)).sum(2)  # noqa: E731
    res = [out, ds @ k * d ** -0.5, share(ds.transpose(-1, -2) @ q * d ** -0.5), share(of_p(p).transpose(-1, -2) @ dout)]
    return [t.transpose(1, 2).to(torch.bfloat16) for t in res]


@pytest.mark.parametrize("b,n,h,kv,d,window,sinks,causal", FEW_KEYS)
def test_one_term_factors_are_noticed(b, n, h, kv, d, window, sinks, causal):
    q, k, v, dout = (rand(b, n, x, d, seed=40 + i, dtype=torch.bfloat16, scale=1.5, dev="cpu")
                     for i, x in enumerate((h, kv, kv, h)))
    rest = (window, sinks, causal)
    valid = torch.ones(b, n, dtype=torch.bool)

    def check(**how):
        check_close(attention(q, k, v, dout, *rest, **how), torch.bfloat16, q, k, v, dout, *rest, valid, d ** -0.5, n)

    two = lambda t: rounded(t) + rounded(t - rounded(t))  # noqa: E731
    check(), check(of_p=two, of_ds=two, of_out=two)
    for mistake in ("of_p", "of_ds", "of_out"):
        with pytest.raises(AssertionError):
            check(**{mistake: rounded})
