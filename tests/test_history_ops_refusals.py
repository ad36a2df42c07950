"""CPU: what the long-history operators refuse, and how -- shapes, sizes and types before any kernel is reached, host
tensors like every other operator, and the C entries by status and message."""
import ctypes
import math

import pytest
import torch


def f32(*shape):
    return torch.zeros(*shape)


ATTENTION = [  # q, k, v, keywords, error, words of its message
    ((2, 5, 4, 32), (2, 5, 3, 32), (2, 5, 3, 32), {}, ValueError, "multiple"),
    ((2, 5, 4, 24), (2, 5, 4, 24), (2, 5, 4, 24), {}, ValueError, "head_dim"),
    ((2, 5, 4, 32), (2, 6, 4, 32), (2, 6, 4, 32), {}, ValueError, "expected"),
    ((2, 5, 4, 32), (2, 5, 4, 32), (2, 5, 2, 32), {}, ValueError, "expected"),
    ((5, 4, 32), (5, 4, 32), (5, 4, 32), {}, ValueError, "expected"),
    ((2, 5, 4, 32), (2, 5, 4, 32), (2, 5, 4, 32), {"window": 0}, ValueError, "window"),
    ((2, 5, 4, 32), (2, 5, 4, 32), (2, 5, 4, 32), {"sinks": -1}, ValueError, "sinks"),
    ((2, 5, 4, 32), (2, 5, 4, 32), (2, 5, 4, 32), {"scale": 0.0}, ValueError, "scale"),
    ((2, 5, 4, 32), (2, 5, 4, 32), (2, 5, 4, 32), {"scale": math.inf}, ValueError, "scale"),
    ((2, 5, 4, 32), (2, 5, 4, 32), (2, 5, 4, 32), {"valid": torch.ones(2, 4, dtype=torch.bool)}, ValueError, "valid"),
    ((2, 5, 4, 32), (2, 5, 4, 32), (2, 5, 4, 32), {"valid": torch.ones(2, 5)}, ValueError, "valid"),
]


@pytest.mark.parametrize("q,k,v,how,error,words", ATTENTION)
def test_window_attention_refusals(asme, q, k, v, how, error, words):
    how = {"window": 3, **how}
    with pytest.raises(error, match=words):
        asme.ops.window_attention(f32(*q), f32(*k), f32(*v), **how)


def test_window_attention_types_and_devices(asme):
    t = f32(1, 2, 1, 16)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        asme.ops.window_attention(t.half(), t.half(), t.half(), 2)
    with pytest.raises(asme._lib.ASMEKernelError, match="no CPU fallback"):
        asme.ops.window_attention(t, t, t, 2)
    for qkv, heads in ((f32(2, 3, 96), 4), (f32(3, 96), 2), (f32(2, 3, 96), 0)):
        with pytest.raises(ValueError):
            asme.ops.window_attention_qkv(qkv, heads, 2)


def test_window_cache_refusals(asme):
    ops = asme.ops
    c, n = f32(2, 2, 10, 32), torch.zeros(2, dtype=torch.int64)
    q, k = f32(2, 4, 32), f32(2, 2, 32)
    for bad in ((f32(2, 10, 32), f32(2, 10, 32)), (c, f32(2, 2, 9, 32)), (f32(2, 2, 10, 24), f32(2, 2, 10, 24)),
                (f32(2, 0, 10, 32), f32(2, 0, 10, 32))):
        with pytest.raises(ValueError):
            ops.window_attention_step(q, k, k, *bad, n)
    for sinks in (-1, 10, 11):
        with pytest.raises(ValueError, match="sinks"):
            ops.window_attention_step(q, k, k, c, c.clone(), n, sinks=sinks)
    with pytest.raises(asme._lib.ASMEKernelError, match="no CPU fallback"):
        ops.window_attention_step(q, k, k, c, c.clone(), n)
    with pytest.raises(asme._lib.ASMEKernelError, match="no CPU fallback"):
        ops.window_cache_fill(c, c.clone(), f32(2, 5, 2, 32), f32(2, 5, 2, 32), n)


@pytest.mark.parametrize("logits,ids,t,tau,error,words", [
    ((3, 7), (3, 2), (3, 3), 1.0, ValueError, "expected"),
    ((3, 7), (2, 2), (2, 2), 1.0, ValueError, "expected"),
    ((3, 7), (3, 0), (3, 0), 1.0, ValueError, "entries"),
    ((3, 7), (3, 1025), (3, 1025), 1.0, ValueError, "entries"),
    ((3, 0), (3, 2), (3, 2), 1.0, ValueError, "item"),
    ((3, 7), (3, 2), (3, 2), 0.0, ValueError, "temperature"),
    ((3, 7), (3, 2), (3, 2), math.inf, ValueError, "temperature"),
    ((3, 7), (3, 2), (3, 2), math.nan, ValueError, "temperature")])
def test_distill_refusals(asme, logits, ids, t, tau, error, words):
    with pytest.raises(error, match=words):
        asme.ops.distill_cross_entropy(f32(*logits), torch.zeros(*ids, dtype=torch.int64), f32(*t), tau)


def test_distill_types(asme):
    op, ids, t = asme.ops.distill_cross_entropy, torch.zeros(3, 2, dtype=torch.int64), f32(3, 2)
    with pytest.raises(TypeError, match="whole"):
        op(f32(3, 7), t, t)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        op(f32(3, 7).double(), ids, t)
    with pytest.raises(ValueError, match="weight"):
        op(f32(3, 7), ids, t, 1.0, math.nan)
    with pytest.raises(ValueError, match="teacher"):
        op(f32(3, 7), ids, t.clone().requires_grad_())
    with pytest.raises(asme._lib.ASMEKernelError, match="no CPU fallback"):
        op(f32(3, 7), ids, t)
    with pytest.raises(ValueError, match="weight"):
        asme.losses.TopKDistillationLoss(weight=1.5)


@pytest.mark.parametrize("res,y,w,how,words", [
    ((2, 3, 8), (2, 3, 9), 8, {}, "differ"),
    ((2, 3, 8), (2, 3, 8), 9, {}, "post_w"),
    ((2, 3, 8), (2, 3, 8), 8, {"pre_w": torch.ones(7)}, "pre_w"),
    ((2, 3, 8), (2, 3, 8), 8, {"pre_b": torch.ones(8)}, "pre_b"),
    ((2, 3, 8), (2, 3, 8), 8, {"gate": torch.ones(3, 8)}, "gate"),
    ((2, 3, 8), (2, 3, 8), 8, {"gate": torch.ones(1, 3, 8)}, "gate"),
    ((2, 3, 8), (2, 3, 8), 8, {"gate": torch.ones(2, 3, 1)}, "gate"),
    ((2, 3, 8), (2, 3, 8), 8, {"residual_scale": math.inf}, "finite"),
    ((2, 3, 8), (2, 3, 8), 8, {"eps": -1.0}, "eps"),
    ((2, 8193), (2, 8193), 8193, {}, "channels"),
    ((2, 0), (2, 0), 0, {}, "channels")])
def test_gated_residual_norm_refusals(asme, res, y, w, how, words):
    def call():
        asme.ops.gated_residual_norm(f32(*res), f32(*y), torch.ones(w), **how)
    # (a gate of another device or type is found with the tensors on the device; its shape is looked at after that)
    if words in ("gate", "post_w", "pre_w"):
        with pytest.raises((ValueError, asme._lib.ASMEKernelError)):
            call()
    else:
        with pytest.raises(ValueError, match=words):
            call()


def test_model_refusals(asme):
    base = dict(transformer_hidden_size=32, num_transformer_heads=2, num_transformer_layers=1, item_vocab_size=50,
                max_seq_length=10)
    with pytest.raises(ValueError, match="attention dropout"):
        asme.SASRecModel(**base, transformer_dropout=0.1, attention_window=4)
    for bad in (dict(attention_window=0), dict(attention_sinks=2), dict(attention_window=3, attention_sinks=-1)):
        with pytest.raises(ValueError, match="attention_window"):
            asme.SASRecModel(**base, transformer_dropout=0.0, **bad)
    m = asme.SASRecModel(**base, transformer_dropout=0.0)
    with pytest.raises(RuntimeError, match="eval"):
        m.train().decode(torch.zeros(1, dtype=torch.int64), None)
    with pytest.raises(ValueError, match="attention_window"):
        asme.layers.WindowCaches(m._sequence_representation_layer.transformer_layer.transformer_blocks, 1, "cpu")
    # nothing new in a model that asks for nothing
    assert not any("gate" in k for k in m.state_dict())
    g = asme.SASRecModel(**base, transformer_dropout=0.1, transformer_attention_dropout=0.0, attention_window=4,
                         attention_sinks=1, gated_norms=True)
    assert sum("gate" in k for k in g.state_dict()) == 6


def test_c_entries_refuse(asme):
    lib = asme._lib.load()
    one = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(one) + 63) // 64 * 64  # never read: every call below is refused on the host
    strides = (ctypes.c_int64 * 24)(*([16] * 24))

    def refused(rc, words):
        assert rc == -1 and words in lib.asme_mi_last_error(), (rc, lib.asme_mi_last_error())

    def fwd(q=p, b=1, h=1, kv=1, n=4, d=16, w=2, s=0, scale=1.0, dtype=0, st=strides, low=None):
        return lib.asme_window_attention_fwd(q, p, p, p, st, None, b, h, kv, n, d, w, s, 1, scale, dtype, low, None, None)

    refused(fwd(q=None), b"null")
    refused(fwd(st=None), b"null")
    for bad in (dict(b=0), dict(h=3, kv=2), dict(n=0), dict(n=1 << 25), dict(d=24), dict(d=256), dict(w=0), dict(s=-1)):
        refused(fwd(**bad), b"size")
    refused(fwd(scale=-1.0), b"scale")
    refused(fwd(dtype=2), b"dtype")
    refused(fwd(q=p + 4), b"alignment")
    refused(fwd(st=(ctypes.c_int64 * 24)(*([18] * 24))), b"alignment")
    refused(fwd(low=p), b"out_low")
    need = lib.asme_window_attention_bwd_workspace(1, 1, 1, 4, 16, 2, 0, 1, 0)
    assert need >= 16
    refused(lib.asme_window_attention_bwd(p, p, p, p, p, p, p, p, strides, None, 1, 1, 1, 4, 16, 2, 0, 1, 1.0, 0, None, p,
                                          p, need - 1, None), b"workspace")
    assert lib.asme_window_attention_bwd_workspace(1, 1, 1, 4, 24, 2, 0, 1, 0) == 0

    def step(q=p, b=1, h=1, kv=1, d=16, slots=4, s=0, dtype=0, ws=None, nb=0):
        return lib.asme_window_step(q, p, p, p, p, p, b, h, kv, d, slots, s, 1.0, dtype, ws, nb, p, None)

    refused(step(q=None), b"null")
    for bad in (dict(b=0), dict(h=3, kv=2), dict(d=24), dict(slots=2, s=2), dict(slots=0), dict(slots=1 << 50)):
        refused(step(**bad), b"size")
    refused(step(q=p + 2), b"alignment")
    refused(step(dtype=7), b"dtype")
    refused(step(slots=4096), b"workspace")
    refused(lib.asme_window_cache_fill(p, p, 64, 16, 17, 64, 16, 16, p, 1, 4, 1, 16, 4, 0, 0, p, p, None), b"alignment")
    refused(lib.asme_window_cache_fill(p, p, 64, 16, 16, 64, 16, 16, p, 1, 0, 1, 16, 4, 0, 0, p, p, None), b"size")

    def distill(x=p, ld=8, n=2, V=8, top=2, tau=1.0, w=1.0, dtype=0, nb=1 << 20):
        return lib.asme_distill_xent_fwd(x, ld, n, V, p, p, top, tau, w, dtype, p, p, p, nb, p, None)

    refused(distill(x=None), b"null")
    for bad in (dict(ld=7), dict(n=0), dict(V=0), dict(V=1 << 31, ld=1 << 31), dict(top=0), dict(top=1025)):
        refused(distill(**bad), b"size")
    refused(distill(tau=0.0), b"temperature")
    refused(distill(w=math.inf), b"weight")
    refused(distill(nb=8), b"workspace")
    for n, V in ((511, 8192), (512, 4095), (512, 32769)):
        assert lib.asme_distill_xent_grad_supported(n, V, 0) == 0
        refused(lib.asme_distill_xent_fwd_grad(p, V, n, V, p, p, 2, 1.0, 1.0, 0, p, p, p + 16, p, 1 << 30, p, None), b"size")
    assert lib.asme_distill_xent_grad_supported(512, 65536, 1) == 1
    refused(lib.asme_distill_xent_fwd_grad(p, 8192, 512, 8192, p, p, 2, 1.0, 1.0, 0, p, p, p + 4, p, 1 << 30, p, None),
            b"aligned")
    refused(lib.asme_scale_by(p + 4, 8, 0, p, None), b"bad")
    refused(lib.asme_distill_xent_bwd(p, 8, 2, 8, p, 2, 1.0, 1.0, 0, p, p, p, p, p, 8, None), b"must not be")

    def norm(res=p, n=4, d=8, per=1, gate=p, dtype=0, eps=1e-5, pre=None, z=None):
        return lib.asme_gated_residual_norm_fwd(res, p, gate, per, p, None, pre, None, n, d, 1.0, eps, 0, dtype, p, z, p,
                                                None)

    refused(norm(res=None), b"null")
    refused(norm(pre=p), b"z_out")
    for bad in (dict(n=0), dict(d=0), dict(d=8193), dict(per=3), dict(per=8), dict(n=1 << 40)):
        refused(norm(**bad), b"size")
    refused(norm(eps=-1.0), b"eps")
    refused(lib.asme_gated_residual_norm_bwd(p, p, None, 1, p, None, None, 4, 8, 1.0, 0, 0, p, None, p, p, p, None, None,
                                             p, 1 << 20, None), b"dz")
    refused(lib.asme_gated_residual_norm_bwd(p, p, None, 1, p, None, None, 4, 8, 1.0, 0, 0, p, p, None, p, p, None, None,
                                             p, 8, None), b"workspace")
