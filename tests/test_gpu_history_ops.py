"""GPU: the long-history operators against plain implementations in 64 bits.

Tolerances.  u = 2^-24 is fp32's largest relative rounding error, an output of type T is rounded once more (by at most
finfo(T).eps / 2 of its value).  Everything between is fp32: a bound is `c * u * size`, where `size` is the sum of the
absolute values of what is added up (computed in 64 bits beside the result) and c counts the roundings on the longest path:
sums run 8 values in a lane, at most 10 shuffle or LDS levels, then serially over turns; exp2 / log / sqrt / division of the
hardware are good to 2 ulp each."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def near(x, ref, size, c, what=""):
    """every element of x within its store rounding plus c * u * size of ref"""
    assert x.shape == ref.shape, (what, x.shape, ref.shape)
    x64, ref, size = x.detach().double().cpu(), ref.detach().double().cpu(), torch.as_tensor(size).double().cpu()
    assert torch.isfinite(x64).all(), what
    off = (x64 - ref).abs()
    room = torch.finfo(x.dtype).eps / 2 * ref.abs() * (1 + 2 ** -7) + c * U * size + 1e-37
    worst = (off / room).max().item() if off.numel() else 0.0
    assert worst <= 1.0, (what, worst, off.max().item())


def rand(*shape, seed, dtype=torch.float32, scale=1.0, dev="cuda"):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g, dtype=torch.float64) * scale).to(dtype).to(dev)


# ------------------------------------------------------------------------------------------------ distillation
def distill64(x, ids, t, tau):
    """loss, its gradient, q, the rows' p on the catalogue"""
    x, t = x.detach().double().cpu(), t.detach().double().cpu()
    ids = ids.cpu()
    n, V = x.shape
    there = (ids >= 0) & (ids < V)
    p = torch.softmax((t / tau).masked_fill(~there, -math.inf), 1).nan_to_num(0.0)
    logq = torch.log_softmax(x / tau, 1)
    rows = there.any(1)
    terms = torch.where(p > 0, p * (p.clamp(min=1e-300).log() - logq.gather(1, ids.clamp(0, V - 1))), 0.0)
    count = rows.sum()
    loss = tau * tau * terms.sum() / count
    on = torch.zeros_like(x).scatter_add_(1, ids.clamp(0, V - 1), torch.where(there, p, 0.0))
    grad = torch.where(rows[:, None], tau / count * (logq.exp() - on), 0.0)
    return loss, grad, logq.exp(), on, count


def distill_lists(n, V, top, seed, empty=True):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, V, (n, top), generator=g)
    if top > 1:
        ids[:, top // 2] = ids[:, 0]  # an item twice on every list
    kept = torch.randint(1, top + 1, (n, 1), generator=g)
    ids = torch.where(torch.arange(top) < kept, ids, -1)
    if empty and n > 2:
        ids[1] = -1         # a row without a list
        ids[2, -1] = V + 5  # beyond the catalogue: absent
    return ids.cuda(), torch.randn(n, top, generator=g).cuda() * 3


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,V,top,tau", [(1, 1, 1, 1.0), (3, 7, 5, 2.0), (5, 1000, 20, 1.0), (64, 10007, 20, 1.5),
                                         (300, 4097, 1, 0.5), (33, 513, 1024, 4.0), (2, 300001, 64, 1.0),
                                         (1030, 255, 8, 1.0), (512, 4096, 3, 1.0), (515, 5003, 1024, 2.0),
                                         (513, 32768, 7, 1.0), (520, 26747, 50, 2.0), (512, 65536, 2, 1.0)])
def test_distill(asme, dev, dtype, n, V, top, tau):
    x = rand(n, V, seed=1, dtype=dtype, scale=3.0).requires_grad_()
    ids, t = distill_lists(n, V, top, 2)
    loss = asme.ops.distill_cross_entropy(x, ids, t, tau)
    (g,) = torch.autograd.grad(loss, x, torch.tensor(0.75, device=dev))
    want, grad, q, on, count = distill64(x, ids, t, tau)
    m = x.detach().abs().max().item() / tau + math.log(V) + 1  # the size of a log q
    r = t.abs().max().item() * 2 / tau + 4                     # relative roundings of a p
    # a row: sum_j p_j (log p_j - log q_j), p_j off by r u, log q_j by 4 u of its terms; rows: positive sums
    near(loss, want, tau * tau * (m + r) * (r + 8), 8, "loss")
    # q: the exponent's terms, and a positive sum of V / 256 serial adds a lane
    # (where the forward holds the gradient it is rounded before the upstream factor and once more after it)
    twice = 2 ** 24 * torch.finfo(dtype).eps / 2 * 0.75 * grad.abs() if n >= 512 and V >= 4096 else 0.0
    near(g, 0.75 * grad, 0.75 * tau / count * (q * (4 * m + V / 256 + 40) + on * (2 * r + 8)) + twice, 1, "gradient")


def test_distill_rows_apart_and_unaligned(asme, dev):
    """logits that are columns of a wider matrix, starting off a 16-byte boundary"""
    wide = rand(9, 1203, seed=3, dtype=torch.bfloat16)
    x = wide[:, 3:1004].detach().requires_grad_()
    assert x.stride(0) == 1203 and x.data_ptr() % 16
    ids, t = distill_lists(9, 1001, 6, 4)
    loss = asme.ops.distill_cross_entropy(x, ids, t, 1.0)
    (g,) = torch.autograd.grad(loss, x)
    y = x.detach().contiguous().clone().requires_grad_()
    other = asme.ops.distill_cross_entropy(y, ids, t, 1.0)
    (h,) = torch.autograd.grad(other, y)
    want, grad, q, on, count = distill64(x, ids, t, 1.0)
    near(loss, want, 40 * 40, 8, "loss")
    near(g, grad, (q + on) / count * 120, 1, "gradient")
    near(h, grad, (q + on) / count * 120, 1, "gradient of the contiguous copy")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_distill_backward_again(asme, dev, dtype):
    """the gradient that a forward already holds is given away once; a second backward of it forms its own"""
    x = rand(600, 4100, seed=3, dtype=dtype).requires_grad_()
    ids, t = distill_lists(600, 4100, 6, 4)
    loss = asme.ops.distill_cross_entropy(x, ids, t, 1.0)
    (a,) = torch.autograd.grad(loss, x, retain_graph=True)
    a.add_(1.0)  # (the caller's own by now)
    (b,) = torch.autograd.grad(loss, x, torch.tensor(2.0, device=dev), retain_graph=True)
    (c,) = torch.autograd.grad(asme.ops.distill_cross_entropy(x, ids, t, 1.0), x, torch.tensor(2.0, device=dev))
    want, grad, q, on, count = distill64(x, ids, t, 1.0)
    size = (q * 200 + on * 40) / count
    near(b, 2 * grad, 2 * size, 1, "second backward")
    # (scaled after it was rounded once: two roundings of the type)
    near(c, 2 * grad, 2 * size + (2 ** 24 * torch.finfo(dtype).eps / 2) * 2 * grad.abs(), 1, "scaled")
    with torch.no_grad():
        x.mul_(1.0)  # a change of the logits in between is noticed, as for every operator
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(loss, x)


def test_distill_no_lists_and_masked_items(asme, dev):
    x = rand(4, 50, seed=5).requires_grad_()
    ids = torch.full((4, 3), -1, device=dev)
    loss = asme.ops.distill_cross_entropy(x, ids, torch.zeros(4, 3, device=dev))
    assert torch.isnan(loss)
    (g,) = torch.autograd.grad(loss, x)
    assert (g == 0).all()
    # items the student may not choose (-inf) off the list: q = 0 and no gradient; absent entries may hold anything
    with torch.no_grad():
        x[:, 10:20] = -math.inf
    ids = torch.tensor([[3, 40, -1]] * 4, device=dev)
    t = torch.tensor([[1.0, 0.5, math.nan]] * 4, device=dev)
    loss = asme.ops.distill_cross_entropy(x, ids, t, 2.0)
    (g,) = torch.autograd.grad(loss, x)
    want, grad, q, on, count = distill64(x, ids, t.nan_to_num(0.0), 2.0)
    near(loss, want, 4 * 100, 8, "loss")
    near(g, grad, (q + on) / count * 2 * 60, 1, "gradient")
    assert (g[:, 10:20] == 0).all()


@pytest.mark.parametrize("n,V", [(5, 300), (600, 4100)])
def test_distill_weight(asme, dev, n, V):
    x = rand(n, V, seed=6).requires_grad_()
    ids, t = distill_lists(n, V, 4, 7)
    loss = asme.ops.distill_cross_entropy(x, ids, t, 1.3, weight=-0.3)
    (g,) = torch.autograd.grad(loss, x)
    want, grad, q, on, count = distill64(x, ids, t, 1.3)
    near(loss, -0.3 * want, 40 * 40, 8, "loss")
    near(g, -0.3 * grad, (q + on) / count * 120, 1, "gradient")


def test_distill_against_differences(asme, dev):
    x = rand(3, 40, seed=6).requires_grad_()
    ids, t = distill_lists(3, 40, 4, 7, empty=False)
    (g,) = torch.autograd.grad(asme.ops.distill_cross_entropy(x, ids, t, 1.3), x)
    d = rand(3, 40, seed=8)
    # central differences with h = 2^-5 along a direction, Richardson-extrapolated: truncation ~ h^4 |d|^5-ish < 1e-4,
    # rounding of the loss (< 2 u * 10) over h: < 1e-4
    def at(h):
        with torch.no_grad():
            return (asme.ops.distill_cross_entropy(x + h * d, ids, t, 1.3)
                    - asme.ops.distill_cross_entropy(x - h * d, ids, t, 1.3)).item() / (2 * h)
    slope = (4 * at(2 ** -5) - at(2 ** -4)) / 3
    assert abs(slope - (g * d).sum().item()) < 1e-3


# ------------------------------------------------------------------------------------------------ gated residual norm
def norm64(x, w, b, rms, eps):
    x = x if rms else x - x.mean(-1, keepdim=True)
    x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w
    return x if b is None else x + b


def gated64(res, y, pw, pb, qw, qb, gate, a, eps, rms):
    br = norm64(y, pw, pb, rms, eps)
    s = a * res + (br if gate is None else gate * br)
    return s, (None if qw is None else norm64(s, qw, qb, rms, eps))


NORM_CASES = [  # batch, length, dim, gate
    (1, 1, 1, "none"), (2, 3, 8, "sequence"), (3, 5, 17, "row"), (2, 37, 128, "channel"), (3, 33, 100, "sequence"),
    (1, 50, 132, "channel"), (4, 9, 256, "row"), (5, 7, 300, "sequence"), (2, 11, 520, "none"), (1, 19, 1024, "channel"),
    (2, 6, 1111, "sequence"), (3, 4, 2048, "row"), (2, 5, 4096, "channel"), (2, 3, 5000, "sequence"),
    (2, 3, 4100, "row"), (1, 4, 8192, "channel"), (1, 3, 8191, "row"), (40, 200, 64, "sequence"), (1, 5000, 64, "channel"),
    (2500, 2, 32, "sequence")]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("b,n,d,kind", NORM_CASES)
def test_gated_residual_norm(asme, dev, dtype, rms, b, n, d, kind):
    shape = {"none": None, "channel": (d,), "sequence": (b, 1, d), "row": (b, n, d)}[kind]
    res, y = rand(b, n, d, seed=1, dtype=dtype, scale=2.0), rand(b, n, d, seed=2, dtype=dtype, scale=0.7)
    y = (y.float() + 0.5).to(dtype)
    gate = None if shape is None else rand(*shape, seed=3, dtype=dtype, scale=0.5)
    pw, qw = 1 + rand(d, seed=4, scale=0.2), 1 + rand(d, seed=5, scale=0.2)
    pb, qb = (None, None) if rms else (rand(d, seed=6, scale=0.2), rand(d, seed=7, scale=0.2))
    a, eps = 1.25, 1e-3
    leaves = [t.requires_grad_() for t in (res, y, gate, pw, pb, qw, qb) if t is not None]
    s, z = asme.ops.gated_residual_norm(res, y, pw, pb, qw, qb, gate=gate, residual_scale=a, eps=eps, rms=rms)
    ds, dz = rand(b, n, d, seed=8, dtype=dtype), rand(b, n, d, seed=9, dtype=dtype)
    got = torch.autograd.grad((s, z), leaves, (ds, dz))
    big = [None if t is None else t.detach().double().cpu().requires_grad_() for t in (res, y, gate, pw, pb, qw, qb)]
    br = norm64(big[1], big[3], big[4], rms, eps)
    s64, z64 = gated64(big[0], big[1], big[3], big[4], big[5], big[6], big[2], a, eps, rms)
    want = torch.autograd.grad((s64, z64), [t for t in big if t is not None], (ds.double().cpu(), dz.double().cpu()))
    with torch.no_grad():
        # sizes: x^ = (x - mean) r is off by c u r max|x| (the mean's rounding) beside c u |x^|
        def spread(x):
            m = 0 if rms else x.mean(-1, keepdim=True)
            r = 1 / torch.sqrt((x - m).square().mean(-1, keepdim=True) + eps)
            return r, 1 + r * x.abs().amax(-1, keepdim=True)
        ry, ey = spread(big[1])
        rs, es = spread(s64)
        g = 1.0 if gate is None else big[2].abs()
        top = lambda t: t.abs().amax(-1, keepdim=True)  # noqa: E731
        w1, w2 = big[3].abs().max(), big[5].abs().max()
        size_s = a * big[0].abs() + g * (w1 * ey + 1)
        size_z = w2 * rs * size_s.amax(-1, keepdim=True) * es + 1
        near(s, s64, size_s, 32, "s")
        near(z, z64, size_z, 64, "z")
        # d = ds + r (h - mean h - x^ mean(h x^)), h = dz w: x^ off as above (relative to `es`, and to s's own error)
        zs = rs * size_s.amax(-1, keepdim=True) + es
        size_d = ds.double().cpu().abs() + rs * w2 * top(dz.double().cpu()) * es * es * zs
        size_d = size_d.expand_as(s64)
        names = ["res", "y"] + ([] if gate is None else ["gate"])
        size_n = (size_d * g).amax(-1, keepdim=True) * w1
        sizes = {"res": a * size_d, "y": (ry * size_n * ey * ey * ey).expand_as(s64)}
        if gate is not None:
            lead = {"channel": (0, 1), "sequence": (1,), "row": ()}[kind]
            size_b = size_d * (w1 * ey + 1)
            sizes["gate"] = size_b.sum(lead).reshape(gate.shape) if lead else size_b
        k = 0
        for name in names:
            near(got[k], want[k], sizes[name], 128, "gradient of " + name)
            k += 1
        # column sums: the rows' sizes added up, and a serial sum's rounding on top (the factor's log-free part: a row
        # lane adds at most rows / 16 terms, partial rows 64 more)
        depth = 128 + b * n / 16
        cols = [(size_d * g * ey).sum((0, 1))] + ([] if rms else [(size_d * g).sum((0, 1))])
        cols += [(dz.double().cpu().abs() * zs * es).sum((0, 1))] + ([] if rms else [dz.double().cpu().abs().sum((0, 1))])
        for c in cols:
            near(got[k], want[k], c, depth, f"column sum {k}")
            k += 1
        assert k == len(got)


def test_gated_residual_norm_parts(asme, dev):
    """one output alone, no second norm, half-precision weights, non-contiguous rows, a gate of one row"""
    res, y = rand(4, 6, 96, seed=1)[:, ::2], rand(3, 4, 96, seed=2).transpose(0, 1)
    w = (1 + rand(96, seed=3, scale=0.1)).to(torch.bfloat16).requires_grad_()
    gate = rand(1, 1, 96, seed=4)
    full = lambda **k: asme.ops.gated_residual_norm(res, y, w, gate=gate, **k)  # noqa: E731
    s, z = full()
    assert z is None
    (g,) = torch.autograd.grad(s, w, torch.ones_like(s))
    assert g.dtype == torch.bfloat16
    big = [t.detach().double().cpu() for t in (res, y, w, gate)]
    s64, _ = gated64(big[0], big[1], big[2], None, None, None, big[3], 1.0, 1e-5, False)
    near(s, s64, 8 + s64.abs(), 32, "s")
    want = (big[3] * norm64(big[1], 1.0, None, False, 1e-5)).sum((0, 1))
    near(g, want, (big[3].abs() * 4 * 12).sum((0, 1)), 64, "gradient of w")
    # z alone: s's gradient is absent
    q = torch.ones(96, device=dev)
    y2 = y.detach().contiguous().requires_grad_()
    s, z = asme.ops.gated_residual_norm(res, y2, w, pre_w=q, gate=gate)
    (a,) = torch.autograd.grad(z, y2, res)
    s, z = asme.ops.gated_residual_norm(res, y2, w, pre_w=q, gate=gate)
    (b,) = torch.autograd.grad((s, z), y2, (torch.zeros_like(s), res.contiguous()))
    assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------ the ring cache
def ring(p, sinks, window):
    return p if p < sinks else sinks + (p - sinks) % window


STEP_CASES = [  # batch, heads, kv_heads, head_dim, window, sinks
    (1, 1, 1, 16, 1, 0), (2, 2, 2, 64, 5, 2), (3, 6, 2, 32, 33, 1), (2, 8, 1, 128, 130, 4), (1, 11, 1, 64, 70, 0),
    (2, 4, 4, 128, 700, 13), (1, 2, 1, 16, 2000, 3), (1, 16, 2, 64, 1023, 1), (65, 3, 3, 32, 20, 0)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,h,kv,d,window,sinks", STEP_CASES)
def test_window_attention_step(asme, dev, dtype, b, h, kv, d, window, sinks):
    slots = window + sinks
    q, k, v = (rand(b, x, d, seed=i, dtype=dtype, scale=1.5) for i, x in ((1, h), (2, kv), (3, kv)))
    ck, cv = (rand(b, kv, slots, d, seed=i, dtype=dtype, scale=1.5) for i in (4, 5))
    g = torch.Generator().manual_seed(6)
    n = torch.randint(0, 3 * slots, (b,), generator=g)
    n[0] = [0, slots - 1, slots, 10 ** 12][d % 4 if d % 4 else (window % 4)]
    if b > 2:
        n[1], n[2] = 0, -1  # the first token; a sequence that takes no step
    for u in range(b):  # what no position has been stored in may hold anything
        held = max(0, min(int(n[u]), slots))
        ck[u, :, held:], cv[u, :, held:] = math.nan, math.inf
    before = ck.clone(), cv.clone()
    out = asme.ops.window_attention_step(q, k, v, ck, cv, n.cuda(), sinks=sinks)
    want, size = torch.zeros(b, h, d, dtype=torch.float64), torch.zeros(b, h, d, dtype=torch.float64)
    for u in range(b):
        if n[u] >= 0:
            to = ring(int(n[u]), sinks, window)
            before[0][u, :, to], before[1][u, :, to] = k[u], v[u]
            held = min(int(n[u]) + 1, slots)
            for i in range(h):
                kk = before[0][u, i // (h // kv), :held].double().cpu()
                vv = before[1][u, i // (h // kv), :held].double().cpu()
                qq = q[u, i].double().cpu() / math.sqrt(d)
                p = torch.softmax(kk @ qq, 0)
                want[u, i] = p @ vv
                # a score is off by (16 + log2 64) u of its terms, a weight by twice that; sums: held / 16 serial adds
                size[u, i] = (p @ vv.abs()) * (2 * 24 * (kk.abs() @ qq.abs()).max() + held / 16 + 32)
    near(out, want, size, 1, "out")
    for got, ref in zip((ck, cv), before):
        assert torch.equal(got.view(torch.int16), ref.view(torch.int16)), "the cache beside the new slot"


@pytest.mark.parametrize("odd", [0, 1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_window_attention_step_stores_at_every_slot(asme, dev, dtype, odd):
    """the slots of a sequence are cut over workgroups: the new token is stored once, whichever of them it falls to"""
    b, d, slots = 261, 64, 521
    k, v, q = (rand(b, 1, d, seed=i, dtype=dtype) for i in (1, 2, 3))
    ck, cv = (rand(b, 1, slots, d, seed=i, dtype=dtype) for i in (4, 5))
    n = 2 * torch.arange(b) + odd + 521  # the ring has come round once
    want = ck.clone(), cv.clone()
    for u in range(b):
        to = ring(int(n[u]), 3, slots - 3)
        want[0][u, :, to], want[1][u, :, to] = k[u], v[u]
    for _ in range(3):
        asme.ops.window_attention_step(q, k, v, ck, cv, n.cuda(), sinks=3)
        assert torch.equal(ck, want[0]) and torch.equal(cv, want[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,n,kv,d,window,sinks", [(1, 1, 1, 16, 1, 0), (3, 9, 2, 32, 4, 2), (4, 50, 1, 64, 16, 5),
                                                   (2, 20, 3, 128, 64, 1), (5, 130, 2, 16, 31, 0)])
def test_window_cache_fill(asme, dev, dtype, b, n, kv, d, window, sinks):
    wide = rand(b, n, 2 * kv, d, seed=1, dtype=dtype)
    k, v = wide[:, :, :kv], wide[:, :, kv:]  # views of one projection's output
    ck, cv = (rand(b, kv, window + sinks, d, seed=i, dtype=dtype) for i in (2, 3))
    g = torch.Generator().manual_seed(4)
    lengths = torch.randint(0, n + 1, (b,), generator=g)
    lengths[-1] = n
    want = ck.clone(), cv.clone()
    for u in range(b):
        for p in range(int(lengths[u])):
            want[0][u, :, ring(p, sinks, window)], want[1][u, :, ring(p, sinks, window)] = k[u, p], v[u, p]
    asme.ops.window_cache_fill(ck, cv, k, v, lengths.cuda(), sinks=sinks)
    assert torch.equal(ck, want[0]) and torch.equal(cv, want[1])


# ------------------------------------------------------------------------------------------------ window attention
def seen64(n, window, sinks, causal, valid):
    i, j = torch.arange(n)[:, None], torch.arange(n)[None]
    if causal:
        m = ((i - j < window) | (j < sinks)) & (j <= i)
    else:
        m = ((i - j).abs() < window) | (j < sinks)
    return m[None] & valid[:, None, :] & valid[:, :, None]


def window64(q, k, v, dout, window, sinks, causal, valid, scale):
    """out, dq, dk, dv in 64 bits, and for each the size that its error is counted in"""
    q, k, v, dout = (t.detach().double().cpu().transpose(1, 2) for t in (q, k, v, dout))
    group = q.shape[1] // k.shape[1]
    ok = valid[:, None, :, None]
    q, k, v, dout = (torch.where(ok, t, 0.0) for t in (q, k, v, dout))
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    m = seen64(q.shape[2], window, sinks, causal, valid)[:, None]
    kt, vt = k.transpose(-1, -2), v.transpose(-1, -2)
    s = (q @ kt * scale).masked_fill(~m, -math.inf)
    p = torch.softmax(s, -1).nan_to_num(0.0)
    out = p @ v
    dp = dout @ vt
    delta = (dout * out).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    share = lambda t: t.unflatten(1, (-1, group)).sum(2)  # noqa: E731
    res = [out, ds @ k * scale, share(ds.transpose(-1, -2) @ q * scale), share(p.transpose(-1, -2) @ dout)]
    # a score is off by es u (its products' terms, one rounding per added k step), so p by a factor 1 + 2 es u;
    # dP and D by 24 u of their terms
    a = scale * (q.abs() @ kt.abs()) * m
    es = 2 * (24 * a.amax(-1, keepdim=True) + 16)
    dps = (dout.abs() @ vt.abs() + (dout.abs() * (p @ v.abs())).sum(-1, keepdim=True)) * m
    dss = p * (dps * (24 + 2 * es))
    sizes = [es * (p @ v.abs()), dss @ k.abs() * scale, share(dss.transpose(-1, -2) @ q.abs() * scale),
             share((p * es).transpose(-1, -2) @ dout.abs())]
    # terms of the sums over keys and queries, for sums of rounded (bf16) weights
    terms = [p @ v.abs(), (ds.abs() @ k.abs()) * scale, share(ds.abs().transpose(-1, -2) @ q.abs() * scale),
             share(p.transpose(-1, -2) @ dout.abs())]
    # what the rounding of the saved output adds to D, and so to dS = P (dP - D)
    half = (dout.abs() * out.abs()).sum(-1, keepdim=True) * p
    more = [torch.zeros_like(out), half @ k.abs() * scale, share(half.transpose(-1, -2) @ q.abs() * scale), 0 * res[3]]
    return tuple([t.transpose(1, 2) for t in x] for x in (res, sizes, terms, more))


def check_window(got, dtype, q, k, v, dout, window, sinks, causal, valid, scale, n):
    res, sizes, terms, more = window64(q, k, v, dout, window, sinks, causal, valid, scale)
    for x, ref, size, term, extra, name in zip(got, res, sizes, terms, more, ("out", "dq", "dk", "dv")):
        # sums over n keys or queries: n / 16 products in a row on an accumulator
        room = size + (n / 16 + 32) * term
        if dtype == torch.bfloat16:
            # P and dS rounded to bf16, the output that D is formed from too: bf16 keeps 8 significant bits, so half a
            # step is at most 2^-8 = 2^16 u of the value (1 + 2^-8 <= x < 1 + 2^-7 rounds by up to 2^-8)
            room = room + 2.0 ** 16 * (term * (1 + 2 ** -6) + extra)
        near(x, ref, room, 1, name)
        assert (x[~valid.to(x.device)] == 0).all(), name


WINDOW_CASES = [  # batch, length, heads, kv_heads, head_dim, window, sinks, causal, padding
    (1, 1, 1, 1, 16, 1, 0, True, False), (2, 3, 2, 1, 32, 2, 1, True, True), (3, 50, 2, 2, 32, 16, 1, True, True),
    (2, 64, 4, 2, 64, 64, 0, True, False), (2, 65, 2, 2, 128, 7, 3, True, True), (1, 200, 3, 1, 64, 64, 2, True, False),
    (2, 257, 2, 2, 16, 31, 40, True, True), (1, 300, 2, 1, 128, 1000, 0, True, True),
    (1, 700, 4, 1, 32, 130, 70, True, True), (2, 200, 2, 2, 64, 33, 5, False, True), (1, 513, 3, 3, 32, 1, 0, False, False),
    (2, 70, 4, 4, 128, 5, 66, False, True), (1, 530, 4, 2, 64, 100, 13, False, True),
    (1, 1200, 2, 1, 64, 5, 1, True, False), (1, 1031, 8, 1, 128, 257, 300, True, True),
    (70, 17, 1, 1, 16, 4, 2, True, True)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,n,h,kv,d,window,sinks,causal,padding", WINDOW_CASES)
def test_window_attention(asme, dev, dtype, b, n, h, kv, d, window, sinks, causal, padding):
    g = torch.Generator().manual_seed(1)
    valid = torch.ones(b, n, dtype=torch.bool)
    if padding:  # right padding, a hole, and (of several) a sequence with nothing in it
        valid = torch.arange(n) < torch.randint(1, n + 1, (b, 1), generator=g)
        valid[:, n // 3] = False
        if b > 1:
            valid[1] = False
    q, k, v, dout = (rand(b, n, x, d, seed=i, dtype=dtype, scale=1.5) for i, x in ((2, h), (3, kv), (4, kv), (5, h)))
    for t, junk in ((q, math.nan), (k, math.inf), (v, math.nan), (dout, -math.inf)):
        t[~valid.cuda()] = junk  # padding may hold anything
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    out = asme.ops.window_attention(q, k, v, window, sinks=sinks, causal=causal,
                                    valid=valid.cuda() if padding else None)
    got = [out, *torch.autograd.grad(out, (q, k, v), dout)]
    check_window(got, dtype, q, k, v, dout, window, sinks, causal, valid, d ** -0.5, n)


# ------------------------------------------------------------------------------------------------ streams and graphs
def history_call(asme, kind, dtype, seed):
    """(inputs to be refilled, a call of them that returns everything it computes)"""
    ops = asme.ops
    if kind == "attention":
        q, k, v, dout = (rand(2, 150, x, 32, seed=seed + i, dtype=dtype) for i, x in enumerate((4, 2, 2, 4)))
        valid = (torch.arange(150) < torch.tensor([[150], [70]])).cuda()
        for t in (q, k, v):
            t.requires_grad_()

        def call():
            out = ops.window_attention(q, k, v, 20, sinks=3, valid=valid)
            return [out, *torch.autograd.grad(out, (q, k, v), dout)]
        return [q, k, v, dout], call
    if kind == "step":
        q, k, v = rand(3, 4, 32, seed=seed, dtype=dtype), rand(3, 2, 32, seed=seed + 1, dtype=dtype), rand(3, 2, 32, seed=seed + 2, dtype=dtype)
        ck, cv = rand(3, 2, 600, 32, seed=seed + 3, dtype=dtype), rand(3, 2, 600, 32, seed=seed + 4, dtype=dtype)
        n = torch.tensor([5, 700, 1300]).cuda()

        def call():
            return [ops.window_attention_step(q, k, v, ck, cv, n, sinks=2), ck.clone(), cv.clone()]
        return [q, k, v, ck, cv], call
    if kind == "distill":
        x = rand(20, 5003, seed=seed, dtype=dtype).requires_grad_()
        ids, t = distill_lists(20, 5003, 9, 3)

        def call():
            loss = ops.distill_cross_entropy(x, ids, t, 2.0)
            return [loss, *torch.autograd.grad(loss, x)]
        return [x], call
    res, y, gate = rand(3, 40, 72, seed=seed, dtype=dtype), rand(3, 40, 72, seed=seed + 1, dtype=dtype), rand(3, 1, 72, seed=seed + 2, dtype=dtype)
    w, b = 1 + rand(72, seed=5, scale=0.1), rand(72, seed=6, scale=0.1)
    ds = rand(3, 40, 72, seed=seed + 3, dtype=dtype)
    leaves = [t.requires_grad_() for t in (res, y, gate, w, b)]

    def call():
        s, z = ops.gated_residual_norm(res, y, w, b, w, b, gate=gate)
        return [s, z, *torch.autograd.grad((s, z), leaves, (ds, ds))]
    return [res, y, gate, ds], call


KINDS = ["attention", "step", "distill", "norm"]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", KINDS)
def test_captured_and_replayed(asme, dev, kind, dtype):
    """two graphs of one call on other inputs, replayed in turn with eager calls in between: each replay gives what an
    eager call gives (the same kernels in the same order: the same bits)"""
    (in1, call1), (in2, call2) = history_call(asme, kind, dtype, 10), history_call(asme, kind, dtype, 50)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            call1(), call2()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for call in (call1, call2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    for turn in range(4):
        for (g, out), ins, call in zip(graphs, (in1, in2), (call1, call2)):
            with torch.no_grad():
                for i, t in enumerate(ins):
                    t.copy_(rand(*t.shape, seed=100 * turn + i, dtype=dtype))
            g.replay()
            torch.cuda.synchronize()
            got = [t.detach().clone() for t in out]
            with torch.no_grad():
                for i, t in enumerate(ins):
                    t.copy_(rand(*t.shape, seed=100 * turn + i, dtype=dtype))
            for a, b in zip(got, call()):
                assert torch.equal(a, b), (kind, turn)


@pytest.mark.parametrize("kind", KINDS)
def test_on_another_stream_and_in_any_order(asme, dev, kind):
    """calls in flight on two streams at once, and again one after the other: the same bits"""
    (_, call1), (_, call2) = history_call(asme, kind, torch.float32, 10), history_call(asme, kind, torch.float32, 50)
    want = [t.detach().clone() for t in call1()], [t.detach().clone() for t in call2()]
    side = torch.cuda.Stream()
    for _ in range(5):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            b = call2()
        a = call1()
        torch.cuda.current_stream().wait_stream(side)
        for got, ref in zip((a, b), want):
            assert all(torch.equal(x, y) for x, y in zip(got, ref))
        torch.cuda.synchronize()
