"""CPU: further refusals of the long-history operators and what they do before any kernel is reached."""
import ctypes
import math

import pytest
import torch


def test_distill_bwd_again_refuses(asme):
    lib = asme._lib.load()
    one = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(one) + 63) // 64 * 64  # never read: every call is refused on the host

    def call(x=p, n=2, V=8, top=2, tau=1.0, w=1.0, dtype=1, g=p + 64):
        return lib.asme_distill_xent_bwd_again(x, V, n, V, p, top, tau, w, dtype, p, p, p, p, g, None)

    for bad, words in ((dict(x=None), b"null"), (dict(g=p), b"must not be"), (dict(n=0), b"size"), (dict(V=0), b"size"),
                       (dict(top=1025), b"size"), (dict(dtype=2), b"dtype"), (dict(tau=0.0), b"temperature"),
                       (dict(w=math.inf), b"weight")):
        assert call(**bad) == -1 and words in lib.asme_mi_last_error(), (bad, lib.asme_mi_last_error())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("make", [
    lambda t: t(2, 1283)[:, :1280].view(2, 5, 4, 64)[:1],                # one sequence of a buffer with odd rows
    lambda t: t(1283 * 3)[3:1283].view(1, 5, 4, 64),                     # from an odd position on
    lambda t: t(5, 64 * 4 + 1)[:, :256].view(5, 4, 64)[None],            # odd rows
    lambda t: t(4, 5, 64).transpose(0, 1)[None],                         # heads outermost: read in place
    lambda t: t(2, 5, 64, 4).transpose(2, 3),                            # head values apart
    lambda t: t(2, 5, 1, 64).expand(2, 5, 4, 64)])                       # one head for all: read in place
def test_strides_that_the_attention_kernels_take(asme, dtype, make):
    """every (B, L, heads, head_dim) view comes out with rows on 16-byte boundaries, axes of size 1 included"""
    x = make(lambda *n: torch.randn(*n).to(dtype))
    y = asme.ops._strided_heads(x)
    per = 16 // y.element_size()
    assert torch.equal(x, y) and y.stride(3) == 1 and y.data_ptr() % 16 == 0
    assert all(s % per == 0 for s in y.stride()[:3])


@pytest.mark.parametrize("scale", [0.0, -0.1, math.inf, math.nan])
def test_the_step_refuses_the_scales_that_attention_refuses(asme, scale):
    lib = asme._lib.load()
    one = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(one) + 63) // 64 * 64  # never read
    assert lib.asme_window_step(p, p, p, p, p, p, 1, 1, 1, 16, 4, 0, scale, 0, None, 0, p, None) == -1
    assert b"scale" in lib.asme_mi_last_error()
