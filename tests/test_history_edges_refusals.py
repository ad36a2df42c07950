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
