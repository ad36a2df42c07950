"""GPU: the long-history operators where one part of a kernel meets another -- sinks beyond the window's reach, workgroups
of every size, the accuracy that bf16 is meant to have -- and calls at the edge of what is allowed.  The 64-bit forms, the
inputs and the counting of roundings are those of test_gpu_history_ops.py."""
import math

import pytest
import torch
import torch.utils.checkpoint

from test_gpu_history_models import L, V, cloze_batch, histories, model
from test_gpu_history_ops import check_window, distill64, distill_lists, near, rand, ring, window64

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


def check_close(got, dtype, q, k, v, dout, window, sinks, causal, valid, scale, n):
    """check_window's counting for the accuracy that bf16 is meant to have: P, dS and the output that D is formed from are
    each the sum of two bf16 terms.  The first leaves at most 2^-8 of the value and the second at most 2^-8 of that: 2^-16
    = 2^8 u of each term in place of 2^16 u"""
    res, sizes, terms, more = window64(q, k, v, dout, window, sinks, causal, valid, scale)
    for x, ref, size, term, extra, name in zip(got, res, sizes, terms, more, ("out", "dq", "dk", "dv")):
        room = size + (n / 16 + 32) * term
        if dtype == torch.bfloat16:
            room = room + 2.0 ** 8 * (term + extra)
        near(x, ref, room, 1, name)


# (waves of 32 queries a workgroup: eight for heads of 64 and bf16 heads of 128 and four else, halved while all workgroups
# have a CU of their own)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,n,h,kv,d,window,sinks,causal", [
    (33, 200, 4, 2, 64, 4, 2, True), (33, 200, 4, 2, 64, 33, 5, False), (33, 200, 4, 2, 128, 64, 3, True),
    (33, 200, 4, 1, 128, 5, 66, False), (33, 201, 4, 4, 32, 16, 1, True), (70, 135, 2, 1, 16, 7, 0, False),
    (25, 160, 4, 2, 64, 21, 1, True),                                      # four waves of heads of 64
    (3, 700, 4, 2, 64, 50, 9, True), (1, 1100, 4, 1, 128, 300, 2, True),   # two; the second in pieces of key blocks
    (2, 1200, 4, 2, 128, 3, 200, True)])                                   # sinks far behind the window
def test_window_attention_in_workgroups_of_every_size(asme, dev, dtype, b, n, h, kv, d, window, sinks, causal):
    valid = ragged(b, n, 5)
    (q, k, v, dout), got = window_call(asme, dtype, b, n, h, kv, d, window, sinks, causal, valid, seed=20)
    check_window(got, dtype, q, k, v, dout, window, sinks, causal, valid, d ** -0.5, n)
    check_close(got, dtype, q, k, v, dout, window, sinks, causal, valid, d ** -0.5, n)


# few keys and columns: scores are small, and what is left of an error is the factors' own rounding.  test_history_bounds.py
# shows that check_close notices P or dS in one term, or D formed from the rounded output, at these sizes
FEW_KEYS = [(3, 60, 2, 1, 16, 3, 1, True), (40, 130, 4, 2, 16, 2, 0, False), (3, 70, 2, 2, 32, 2, 1, True)]


@pytest.mark.parametrize("b,n,h,kv,d,window,sinks,causal", FEW_KEYS)
def test_window_attention_of_few_keys(asme, dev, b, n, h, kv, d, window, sinks, causal):
    valid = torch.ones(b, n, dtype=torch.bool)
    (q, k, v, dout), got = window_call(asme, torch.bfloat16, b, n, h, kv, d, window, sinks, causal, None, seed=40)
    check_close(got, torch.bfloat16, q, k, v, dout, window, sinks, causal, valid, d ** -0.5, n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,h,d,window,sinks,causal", [(200, 4, 64, 40, 2, True), (130, 4, 128, 9, 1, False),
                                                       (300, 2, 32, 100, 5, True)])
def test_a_sequence_does_not_depend_on_its_batch(asme, dev, dtype, n, h, d, window, sinks, causal):
    """a workgroup's size follows from the batch; what a query sees, the order of its sums and their roundings do not"""
    valid = torch.ones(130, n, dtype=torch.bool)
    valid[:, n - 3:] = False
    (q, k, v, dout), (out, dq, _, _) = window_call(asme, dtype, 130, n, h, h, d, window, sinks, causal, valid)
    one = [t[7:8].detach().clone().requires_grad_() for t in (q, k, v)]
    alone = asme.ops.window_attention(*one, window, sinks=sinks, causal=causal, valid=valid[7:8].cuda())
    (grad,) = torch.autograd.grad(alone, one[0], dout[7:8])
    assert torch.equal(alone[0], out[7]) and torch.equal(grad[0], dq[7])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_sequence_of_a_buffer_with_odd_rows(asme, dev, dtype):
    q, k, v = (rand(2, 1283, seed=i, dtype=dtype)[:, :1280].view(2, 5, 4, 64)[:1].requires_grad_() for i in (1, 2, 3))
    dout = rand(2, 1283, seed=4, dtype=dtype)[:, :1280].view(2, 5, 4, 64)[:1]
    out = asme.ops.window_attention(q, k, v, 3, sinks=1)
    got = [out, *torch.autograd.grad(out, (q, k, v), dout)]
    same = [t.detach().clone(memory_format=torch.contiguous_format).requires_grad_() for t in (q, k, v)]
    other = asme.ops.window_attention(*same, 3, sinks=1)
    for a, b in zip(got, [other, *torch.autograd.grad(other, same, dout)]):
        assert torch.equal(a, b)
    ck = torch.zeros(1, 4, 4, 64, device=dev, dtype=dtype)
    cv, n = torch.zeros_like(ck), torch.tensor([5], device=dev)
    asme.ops.window_cache_fill(ck, cv, k, v, n, sinks=1)
    assert torch.equal(ck[0, :, 1:], k.detach()[0].transpose(0, 1)[:, [4, 2, 3]])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,n", [(0, 5), (3, 0)])
def test_nothing_to_do_has_gradients_too(asme, dev, dtype, b, n):
    """no sequences, or sequences of no positions: outputs of the right shape and type, and a gradient of every input"""
    q, k, v, qkv = (torch.zeros(b, n, *x, device=dev, dtype=dtype, requires_grad=True)
                    for x in ((4, 32), (2, 32), (2, 32), (192,)))
    out, fused = asme.ops.window_attention(q, k, v, 3), asme.ops.window_attention_qkv(qkv, 2, 3)
    assert out.shape == (b, n, 4, 32) and fused.shape == (b, n, 64) and out.dtype == fused.dtype == dtype
    for t, g in zip((q, k, v, qkv), torch.autograd.grad(out.sum() + fused.sum(), (q, k, v, qkv))):
        assert g.shape == t.shape and g.dtype == dtype
    res, y = (torch.zeros(b, n, 8, device=dev, dtype=dtype, requires_grad=True) for _ in range(2))
    gate = torch.full((b, 1, 8), math.inf, device=dev, dtype=dtype, requires_grad=True)
    w = [torch.ones(8, device=dev, requires_grad=True) for _ in range(4)]
    s, z = asme.ops.gated_residual_norm(res, y, *w, gate=gate)
    assert s.shape == z.shape == res.shape and s.dtype == z.dtype == dtype and s is not z
    for t, g in zip((res, y, gate, *w), torch.autograd.grad((s, z), (res, y, gate, *w), (s, z))):
        assert g.shape == t.shape and g.dtype == t.dtype and (g == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale", [0.03, 1.3])
def test_window_attention_takes_a_scale(asme, dev, dtype, scale):
    valid = ragged(3, 150, 7)
    (q, k, v, dout), got = window_call(asme, dtype, 3, 150, 4, 2, 32, 20, 3, True, valid, scale=scale)
    check_close(got, dtype, q, k, v, dout, 20, 3, True, valid, scale, 150)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("causal", [True, False])
def test_window_attention_of_one_projection(asme, dev, dtype, causal):
    """window_attention_qkv, also of a projection whose rows are apart: what separate q, k and v give, bit for bit"""
    b, n, h, d = 3, 130, 4, 64
    wide = rand(b, n, 3 * h * d + 8, seed=3, dtype=dtype, scale=1.5)
    valid, dout = ragged(b, n, 8).cuda(), rand(b, n, h * d, seed=4, dtype=dtype)
    parts = [t.clone().view(b, n, h, d).requires_grad_() for t in wide[..., :3 * h * d].split(h * d, -1)]
    want = asme.ops.window_attention(*parts, 20, sinks=3, causal=causal, valid=valid)
    grads = torch.autograd.grad(want, parts, dout.view(b, n, h, d))
    for qkv in (wide[..., :3 * h * d].contiguous().requires_grad_(), wide[..., :3 * h * d].detach().requires_grad_()):
        out = asme.ops.window_attention_qkv(qkv, h, 20, sinks=3, causal=causal, valid=valid)
        (g,) = torch.autograd.grad(out, qkv, dout)
        assert torch.equal(out, want.reshape(b, n, h * d))
        assert torch.equal(g, torch.cat([t.reshape(b, n, h * d) for t in grads], -1))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_window_attention_of_views(asme, dev, dtype):
    """inputs and an output's gradient in other orders, broadcast ones, and gradients of some inputs alone"""
    b, n, h, d = 2, 90, 4, 32
    q = rand(b, h, n, d, seed=1, dtype=dtype).transpose(1, 2)       # heads outermost
    k = rand(n, b, 2, d, seed=2, dtype=dtype).transpose(0, 1)       # tokens outermost
    v = rand(b, n, 1, d, seed=3, dtype=dtype).expand(b, n, 2, d)    # one value head for all key heads
    dout = rand(d, h, n, b, seed=4, dtype=dtype).permute(3, 2, 1, 0)
    plain = [t.clone(memory_format=torch.contiguous_format) for t in (q, k, v, dout)]

    def grads(q, k, v, dout, which=(0, 1, 2)):
        leaves = [t.detach().requires_grad_(i in which) for i, t in enumerate((q, k, v))]
        out = asme.ops.window_attention(*leaves, 11, sinks=2)
        return [out.detach(), *torch.autograd.grad(out, [leaves[i] for i in which], dout)]

    want = grads(*plain)
    for a, b_ in zip(grads(q, k, v, dout), want):
        assert torch.equal(a, b_)
    for which in ((0,), (1,), (2,), (0, 2)):
        for a, i in zip(grads(q, k, v, dout, which)[1:], which):
            assert torch.equal(a, want[1 + i]), which
    ones = torch.ones((), device=dev, dtype=dtype).expand(b, n, h, d)
    for a, b_ in zip(grads(q, k, v, ones), grads(*plain[:3], torch.ones_like(plain[3]))):
        assert torch.equal(a, b_)
    one = rand(b, n, 1, d, seed=3, dtype=dtype).requires_grad_()  # a broadcast input's gradient is the sum over its copies
    out = asme.ops.window_attention(q, k, one.expand(b, n, 2, d), 11, sinks=2)
    (g,) = torch.autograd.grad(out, one, dout)
    half = want[3].double()
    near(g, half.sum(2, keepdim=True), half.abs().sum(2, keepdim=True), 2, "broadcast v")


def test_window_attention_beyond_32_bit_offsets(asme, dev):
    """tokens so far apart that a sequence spans 2^32 values: the bits of a compact copy"""
    n, h, d, apart = 1100, 2, 32, 1 << 22
    compact = [rand(1, n, h, d, seed=i, dtype=torch.bfloat16) for i in range(1, 5)]

    def spread(t):
        big = torch.empty(n * apart, device=dev, dtype=torch.bfloat16).as_strided((1, n, h, d), (n * apart, apart, d, 1))
        return big.copy_(t)

    def grads(q, k, v, dout):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = asme.ops.window_attention(*leaves, 70, sinks=3)
        return [out, *torch.autograd.grad(out, leaves, dout)]

    for a, b in zip(grads(*map(spread, compact)), grads(*compact)):
        assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------ the ring cache
def cache_calls(asme, dev):
    q, k = rand(2, 4, 32, seed=1), rand(2, 2, 32, seed=2)
    prompt, n = rand(2, 5, 2, 32, seed=3), torch.tensor([4, 9], device=dev)
    return {"step": lambda ck, cv: asme.ops.window_attention_step(q, k, k, ck, cv, n, sinks=1),
            "fill": lambda ck, cv: asme.ops.window_cache_fill(ck, cv, prompt, prompt, n, sinks=1)}


@pytest.mark.parametrize("kind", ["step", "fill"])
def test_changed_caches_are_noticed(asme, dev, kind):
    call = cache_calls(asme, dev)[kind]
    ck, cv = rand(2, 2, 7, 32, seed=4), rand(2, 2, 7, 32, seed=5)
    w = torch.ones(32, device=dev, requires_grad=True)
    for cache in (ck, cv):
        y = (cache * w).sum()
        with torch.no_grad():
            call(ck, cv)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            y.backward()
    with pytest.raises(RuntimeError, match="no gradient"):
        call(ck.clone().requires_grad_(), cv)
    with torch.inference_mode():  # (tensors without a counter)
        a, b = ck.clone(), cv.clone()
        call(a, b)
    call(ck, cv)
    assert torch.equal(a, ck) and torch.equal(b, cv)


def test_the_step_takes_a_scale(asme, dev):
    """and refuses what window_attention refuses"""
    q, k, ck, cv = rand(2, 4, 32, seed=1), rand(2, 2, 32, seed=2), rand(2, 2, 7, 32, seed=4), rand(2, 2, 7, 32, seed=5)
    n = torch.tensor([3, 9], device=dev)
    for scale in (0.0, -0.1, math.inf, math.nan):
        with pytest.raises(ValueError, match="scale"):
            asme.ops.window_attention_step(q, k, k, ck, cv, n, sinks=1, scale=scale)
    got = asme.ops.window_attention_step(q, k, k, ck.clone(), cv.clone(), n, sinks=1, scale=0.5)
    # (a factor that is a power of two rounds nothing, wherever it is applied)
    want = asme.ops.window_attention_step(q * 0.5, k, k, ck, cv, n, sinks=1, scale=1.0)
    assert torch.equal(got, want)


def test_a_cache_beyond_32_bit_offsets(asme, dev):
    """two sequences of 2^26 slots of 64: one token against them, and a prompt laid in, behind the 2^32nd value"""
    d, window, sinks = 64, (1 << 26) - 5, 5
    slots = window + sinks
    ck = torch.zeros(2, 1, slots, d, device=dev, dtype=torch.bfloat16)
    cv = torch.zeros_like(ck)
    q = torch.ones(2, 2, d, device=dev, dtype=torch.bfloat16)
    k, v = q[:, :1] * 0.125, q[:, :1] * 3
    far = slots - 3  # a key whose score is 64 above all others has all of the weight: 2^26 e^-64 of it elsewhere
    ck[:, 0, far], cv[:, 0, far] = 8.0, torch.arange(d, device=dev).to(torch.bfloat16)
    n = torch.tensor([slots - 2, 5 * window + slots - 2], device=dev)
    out = asme.ops.window_attention_step(q, k, v, ck, cv, n, sinks=sinks)
    # (whole numbers up to 63, exact in bf16; what the others add, at most 3 (2^26 e^-64 + e^-63) < 1e-19, is seen at 0 alone)
    assert (out.double() - cv[:, :, far].double()).abs().max() < 1e-18
    for b in range(2):
        to = ring(int(n[b]), sinks, window)
        assert to == slots - 2 and torch.equal(ck[b, 0, to], k[b, 0]) and torch.equal(cv[b, 0, to], v[b, 0])
    ck.zero_()
    prompt = rand(2, 40, 1, d, seed=3, dtype=torch.bfloat16)
    asme.ops.window_cache_fill(ck, cv, prompt, prompt, torch.tensor([40, 0], device=dev), sinks=sinks)
    assert torch.equal(ck[0, 0, :40], prompt[0, :, 0]) and not ck[0, 0, 40:].any() and not ck[1].any()
    assert torch.equal(cv[0, 0, :40], prompt[0, :, 0]) and torch.equal(cv[:, 0, far], torch.arange(
        d, device=dev).to(torch.bfloat16).expand(2, d))


# ------------------------------------------------------------------------------------------------ distillation
@pytest.mark.parametrize("factor", [0.75, 3.0, 1.0, -0.1])
@pytest.mark.parametrize("n,V", [(600, 4100), (513, 40007)])
def test_distill_rounds_a_bf16_gradient_once(asme, dev, n, V, factor):
    """where the forward formed the gradient too, an upstream factor is applied before the one rounding: within half a step
    of the exact gradient, and the bits of a backward that forms its own"""
    x = rand(n, V, seed=3, dtype=torch.bfloat16, scale=2.0).requires_grad_()
    ids, t = distill_lists(n, V, 6, 4)
    f = torch.tensor(factor, device=dev)
    loss = asme.ops.distill_cross_entropy(x, ids, t, 1.5)
    (a,) = torch.autograd.grad(loss, x, f, retain_graph=True)
    (b,) = torch.autograd.grad(loss, x, f)  # (the second one of a forward)
    want, grad, q, on, count = distill64(x, ids, t, 1.5)
    m, r = x.detach().abs().max().item() / 1.5 + math.log(V) + 1, t.abs().max().item() * 2 / 1.5 + 4  # (as in test_distill)
    near(a, factor * grad, abs(factor) * 1.5 / count * (q * (4 * m + V / 256 + 40) + on * (2 * r + 8)), 1, "gradient")
    assert torch.equal(a, b)


@pytest.mark.parametrize("n,V", [(3, 50), (600, 4100)])
def test_distill_does_not_lose_a_nan_of_the_teacher(asme, dev, n, V):
    """a NaN among a row's present logits makes the loss NaN, also where nothing else is on the list; absent entries may
    hold one; a list of -inf alone is empty"""
    x = rand(n, V, seed=5).requires_grad_()
    ids = torch.tensor([[3, 40, -1]] * n, device=dev)
    ids[1] = torch.tensor([7, -1, V])
    t = torch.tensor([[1.0, 0.5, math.nan]] * n, device=dev)
    assert torch.isfinite(asme.ops.distill_cross_entropy(x, ids, t))
    for row, col in ((1, 0), (2, 0), (2, 1)):
        bad = t.clone()
        bad[row, col] = math.nan
        loss = asme.ops.distill_cross_entropy(x, ids, bad)
        (g,) = torch.autograd.grad(loss, x)
        assert torch.isnan(loss) and torch.isnan(g[row, ids[row, col]]), (row, col)
        assert torch.isfinite(g[torch.arange(n, device=dev) != row]).all()
    low = t.clone()
    low[1] = -math.inf
    loss = asme.ops.distill_cross_entropy(x, ids, low)
    (g,) = torch.autograd.grad(loss, x)
    gone = ids.clone()
    gone[1] = -1
    assert torch.equal(loss, asme.ops.distill_cross_entropy(x, gone, t)) and (g[1] == 0).all()


@pytest.mark.parametrize("n,V", [(3, 50), (600, 4100)])
def test_distill_loss_is_added_to_in_place(asme, dev, n, V):
    x = rand(n, V, seed=5).requires_grad_()
    ids, t = distill_lists(n, V, 6, 4)
    loss = asme.ops.distill_cross_entropy(x, ids, t)
    (want,) = torch.autograd.grad(loss, x)
    total = asme.ops.distill_cross_entropy(x, ids, t)
    total += x.square().sum()
    total *= 2
    (g,) = torch.autograd.grad(total, x)
    assert loss.shape == () and torch.equal(total, 2 * (loss + x.square().sum()))
    near(g, 2 * (want.double() + 2 * x.double()), 4 * x.abs() + 4 * want.abs(), 4, "gradient")


@pytest.mark.parametrize("top", [53, 998])
@pytest.mark.parametrize("n,V", [(1, 2000), (512, 4096)])
def test_distill_probabilities_of_a_long_list(asme, dev, n, V, top):
    """equal logits: p is 1 / top, rounded once -- to 2^-24 of it, as the gradient of an item whose own q is nothing"""
    x = torch.zeros(n, V, device=dev)
    x[:, :top] = -60.0
    x.requires_grad_()
    ids = torch.arange(top, device=dev).expand(n, top)
    (g,) = torch.autograd.grad(asme.ops.distill_cross_entropy(x, ids, torch.full((n, top), 1.7, device=dev)), x)
    # (n is a power of two, the factor 1 / n exact; q < e^-60)
    assert ((g[:, :top].double() * n * top + 1).abs() <= 2.0 ** -24 * (1 + 2.0 ** -20)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_distill_saves_its_gradient_where_hooks_see_it(asme, dev, dtype):
    """what the forward keeps goes through saved-tensor hooks: offloaded to the host, or formed again by a checkpoint"""
    n, V = 2048, 4100
    x = rand(n, V, seed=5, dtype=dtype).requires_grad_()
    ids, t = distill_lists(n, V, 6, 4)
    f = torch.tensor(2.5, device=dev)
    (want,) = torch.autograd.grad(asme.ops.distill_cross_entropy(x, ids, t), x, f)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    with torch.autograd.graph.save_on_cpu():
        loss = asme.ops.distill_cross_entropy(x, ids, t)
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() - before < x.numel() * x.element_size() / 4
    (g,) = torch.autograd.grad(loss, x, f, retain_graph=True)
    assert torch.equal(g, want)
    (again,) = torch.autograd.grad(loss, x, f)
    # the first was formed with the forward and scaled, this one formed anew: q rounded (or not, where it is contracted into
    # q - p) before the subtraction on either side, then at most three products each -- up to 8 u of the terms q and p
    _, _, q, on, count = distill64(x, ids, t, 1.0)
    near(again, want, 2.5 / count * (q + on), 8, "again")
    loss = torch.utils.checkpoint.checkpoint(asme.ops.distill_cross_entropy, x, ids, t, use_reentrant=False)
    (g,) = torch.autograd.grad(loss, x, f)
    assert torch.equal(g, want)


class Distilled(torch.nn.Module):
    def __init__(self, asme, ids, t):
        super().__init__()
        self.op = asme.ops.distill_cross_entropy
        self.register_buffer("ids", ids), self.register_buffer("t", t)

    def forward(self, x):
        return self.op(x, self.ids, self.t)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_distill_backward_captured_apart_and_replayed(asme, dev, dtype):
    """a backward with a graph of its own, replayed several times for one replay of the forward's"""
    n, V = 600, 4100
    ids, t = distill_lists(n, V, 6, 4)
    graphed = torch.cuda.make_graphed_callables(Distilled(asme, ids, t), (rand(n, V, seed=5, dtype=dtype).requires_grad_(),))
    for turn in range(3):
        x = rand(n, V, seed=6 + turn, dtype=dtype).requires_grad_()
        loss, eager = graphed(x), asme.ops.distill_cross_entropy(x, ids, t)
        assert torch.equal(loss, eager)
        _, _, q, on, count = distill64(x, ids, t, 1.0)
        for f in (2.0, 1.0, 0.5, 2.0):
            (g,) = torch.autograd.grad(loss, x, torch.tensor(f, device=dev), retain_graph=True)
            (want,) = torch.autograd.grad(eager, x, torch.tensor(f, device=dev), retain_graph=True)
            # (as in the test before)
            near(g.clone(), want, f / count * (q + on), 8 if dtype == torch.float32 else 0, (turn, f))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_distill_captured_with_its_gradient(asme, dev, dtype):
    """forward and backward in one graph where the forward forms the gradient: every replay gives an eager call's bits"""
    n, V = 600, 4100
    x, f = rand(n, V, seed=5, dtype=dtype).requires_grad_(), torch.tensor(2.0, device=dev)
    ids, t = distill_lists(n, V, 6, 4)

    def call():
        loss = asme.ops.distill_cross_entropy(x, ids, t, 2.0)
        return [loss, *torch.autograd.grad(loss, x, f)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for turn, factor in enumerate((2.0, 1.0, 0.3, 1.0)):
        with torch.no_grad():
            x.copy_(rand(n, V, seed=20 + turn, dtype=dtype)), f.fill_(factor)
        graph.replay()
        graph.replay()
        torch.cuda.synchronize()
        got = [o.detach().clone() for o in out]
        for a, b in zip(got, call()):
            assert torch.equal(a, b), turn


# ------------------------------------------------------------------------------------------------ training and serving
@pytest.mark.parametrize("weight", [0.0, 0.3, 1.0])
def test_training_on_batches_without_lists(asme, dev, weight):
    """a batch in which no row has a list has the cross-entropy alone; a teacher's NaN is no missing list"""
    m = model(asme, "BERT4RecModel", attention_window=6, attention_sinks=1)
    train = asme.MaskedTrainingModule(model=m, item_tokenizer=asme.tokenization.Tokenizer(V - 3), metrics=None)
    batch = cloze_batch(asme, 6, 11)
    loss = train.training_step(dict(batch), 0)["loss"]
    names, leaves = zip(*m.named_parameters())
    want = dict(zip(names, torch.autograd.grad(loss, leaves, allow_unused=True)))
    train.distillation = asme.losses.TopKDistillationLoss(temperature=2.0, weight=weight)
    for ids, logits in ((-1, 0.0), (V, 0.0), (5, -math.inf)):
        none = {**batch, "teacher.ids": torch.full_like(batch["teacher.ids"], ids),
                "teacher.logits": torch.full_like(batch["teacher.logits"], logits)}
        mixed = train.training_step(none, 0)["loss"]
        # (fused logits and cross-entropy there, logits first here: a few roundings of O(1) terms)
        assert abs(mixed.item() - (1 - weight) * loss.item()) < 1e-5 * loss.item()
        for name, g in zip(names, torch.autograd.grad(mixed, leaves, allow_unused=True)):
            assert (g is None) == (want[name] is None), name
            if g is not None:  # (the keys' bias: what the roundings leave of a sum of terms as large as the weights')
                size = want[name.replace("bias", "weight") if name.endswith("linear_layers.1.bias") else name]
                assert (g - (1 - weight) * want[name]).abs().max() <= 5e-5 * size.abs().max().clamp(min=1e-3), name
    if weight:
        batch["teacher.logits"] = batch["teacher.logits"].clone()
        batch["teacher.ids"][:, 0, 0] = 5
        batch["teacher.logits"][:, 0, 0] = math.nan
        assert torch.isnan(train.training_step(batch, 0)["loss"])


def test_prefill_of_a_user_without_history(asme, dev):
    """zeros for that user, nothing else changed, and its first items decoded from an empty cache"""
    m = model(asme, attention_window=5, attention_sinks=1).eval()
    seq, lengths = histories(asme, 4, 9, 5)
    want, _ = m.prefill(seq)
    mask = seq.padding_mask.clone()
    mask[1:3] = False
    rep, caches = m.prefill(asme.InputSequence(seq.sequence * mask, mask))
    assert (rep[1:3] == 0).all() and torch.equal(rep[[0, 3]], want[[0, 3]])
    assert caches.lengths.tolist() == [9, 0, 0, int(lengths[3])]
    whole = torch.zeros(4, L, dtype=torch.int64, device=dev)
    whole[:, :9] = seq.sequence * mask
    for t in range(7):
        items = torch.tensor([3 + t, 20 + t, 40 - t, 7], device=dev)
        whole[torch.arange(4), caches.lengths] = items
        rep = m.decode(items, caches)
        mask = torch.arange(L, device=dev) < caches.lengths[:, None]
        with torch.no_grad():
            want = m.encode(asme.InputSequence(whole, mask))[torch.arange(4), caches.lengths - 1]
        assert (rep - want).abs().max() < 2e-5 * want.abs().max(), t  # (as in test_gpu_history_models.py)
    nobody = torch.zeros_like(mask)
    rep, caches = m.prefill(asme.InputSequence(whole * 0, nobody))
    assert (rep == 0).all() and caches.most == 0


def test_hooks_on_every_norm_of_gated_blocks_run(asme, dev):
    """norms with forward hooks are called as modules, and what a hook returns is used"""
    m = model(asme, attention_window=5, attention_sinks=1, gated_norms=True).eval()
    seq, _ = histories(asme, 4, L, 5)
    layer = m._sequence_representation_layer.transformer_layer
    norms = {n: x for n, x in layer.named_modules() if isinstance(x, torch.nn.LayerNorm)}
    assert len(norms) == 8
    with torch.no_grad():
        want = m.encode(seq)
        for name, norm in norms.items():
            seen = []
            handle = norm.register_forward_hook(lambda mod, args, out: seen.append(out.clone()))
            got = m.encode(seq)
            handle.remove()
            # (another kernel's order of sums in two blocks: a few hundred roundings of O(1) terms)
            assert len(seen) == 1 and (got - want).abs().max() < 2e-5 * want.abs().max(), name
            handle = norm.register_forward_hook(lambda mod, args, out: out * 0.5)
            half = m.encode(seq)
            handle.remove()
            norm.weight.mul_(0.5), norm.bias.mul_(0.5)
            assert (half - m.encode(seq)).abs().max() < 2e-5 * half.abs().max(), name
            norm.weight.mul_(2.0), norm.bias.mul_(2.0)
