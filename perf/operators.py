"""The long-history operators as cases: sliding-window attention with sinks (training, prompt, one new token), the
distillation loss over a teacher's best items, and the gated residual between two norms.

`run` computes a case in its plain form (elementary torch operations in 32 bits) or, with `own` true, through the
package's operators; `exact` computes it from the definitions in 64 bits."""
import math

import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def _ops():
    import __graft_entry__

    return __graft_entry__.load_package().ops


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one optimiser step's attention of a small model on short sessions: launches, not work
        _attention("attention_small", "float32", 4, 50, 2, 2, 32, 16, 1, True, True),
        # the session length and width this package trains at (L = 200, d = 128 in two heads), padded histories
        _attention("attention_session", "float32", 256, 200, 2, 2, 64, 64, 2, True, True),
        # a user's whole history in bfloat16, four query heads to a key head
        _attention("attention_history", "bfloat16", 2, 8192, 16, 4, 128, 1024, 4, True, False),
        # cloze training reads both directions; lengths that fit no tile
        _attention("attention_cloze", "float32", 3, 2049, 6, 2, 64, 257, 5, False, True),
        # ragged prompts: their attention, and what later tokens need of them laid into the cache
        _serving("prompt", "prompt_ragged", "bfloat16", 8, 2000, 8, 2, 64, 512, 8),
        # one user's next item: latency
        _serving("step", "step_single", "float32", 1, 1, 2, 2, 64, 128, 2),
        # a full server: every user's next item over long windows
        _serving("step", "step_batch", "bfloat16", 64, 1, 32, 8, 128, 4096, 4),
        # a few masked positions over an odd catalogue
        _distill("distill_few", "bfloat16", 64, 10007, 20, 1.0),
        # the masked positions of a training batch over the ml-20m catalogue
        _distill("distill_catalogue", "float32", 8192, 26747, 50, 2.0),
        # one short session through a block's end
        _norm("norm_small", "float32", 2, 37, 128, "none", 1.0, False),
        # the training batch's rows, each user's gate on all of the user's rows
        _norm("norm_session", "float32", 1024, 200, 128, "sequence", 1.0, False),
        # wide rows in bfloat16, a gate for each channel and a scaled residual, root-mean-square norms
        _norm("norm_wide", "bfloat16", 4, 4096, 4096, "channel", 1.25, True),
    ]


def draw(rng):
    def spread(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    kind = rng.choice(["attention", "attention", "prompt", "step", "step", "distill", "distill", "norm", "norm"])
    dtype = rng.choice(["float32", "bfloat16"])
    if kind in ("attention", "prompt"):
        while True:
            kv, group, dim = rng.choice([1, 2, 3, 4]), rng.choice([1, 1, 2, 4]), rng.choice([16, 32, 64, 128])
            b, length, window = spread(1, 256), spread(2, 8192), spread(4, 2048)
            if b * kv * group * length * length * dim <= 2 * 16 * 8192 * 8192 * 64:
                break
        sinks = rng.choice([0, 1, 4, 13])
        if kind == "prompt":
            return _serving("prompt", None, dtype, b, length, kv * group, kv, dim, window, sinks)
        return _attention(None, dtype, b, length, kv * group, kv, dim, window, sinks, rng.random() < 0.6,
                          rng.random() < 0.6)
    if kind == "step":
        while True:
            kv, group, dim = rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 2, 4, 8]), rng.choice([16, 32, 64, 128])
            b, window = spread(1, 256), spread(16, 16384)
            if b * kv * window * dim <= 64 * 8 * 4096 * 64:
                break
        return _serving("step", None, dtype, b, 1, kv * group, kv, dim, window, rng.choice([0, 1, 4, 13]))
    if kind == "distill":
        while True:
            n, items = spread(4, 8192), spread(100, 400000)
            if n * items <= 8192 * 26747:
                break
        return _distill(None, dtype, n, items, min(items, spread(1, 256)), rng.choice([1.0, 2.0, 3.5]))
    while True:
        b, length, dim = spread(1, 1024), spread(1, 4096), spread(8, 8192)
        if b * length * dim <= 4 * 4096 * 4096 // 2:
            break
    return _norm(None, dtype, b, length, dim, rng.choice(["none", "channel", "sequence", "row"]),
                 rng.choice([1.0, 0.7]), rng.random() < 0.5)


def _named(name, case):
    return dict(case, name=name) if name else case


def _attention(name, dtype, b, length, heads, kv, dim, window, sinks, causal, ragged):
    return _named(name, {"kind": "attention", "dtype": dtype, "batch": b, "length": length, "heads": heads,
                         "kv_heads": kv, "head_dim": dim, "window": window, "sinks": sinks, "causal": causal,
                         "ragged": ragged})


def _serving(kind, name, dtype, b, length, heads, kv, dim, window, sinks):
    return _named(name, {"kind": kind, "dtype": dtype, "batch": b, "length": length, "heads": heads, "kv_heads": kv,
                         "head_dim": dim, "window": window, "sinks": sinks})


def _distill(name, dtype, rows, items, top, temperature):
    return _named(name, {"kind": "distill", "dtype": dtype, "rows": rows, "items": items, "top": top,
                         "temperature": temperature})


def _norm(name, dtype, b, length, dim, gate, residual_scale, rms):
    return _named(name, {"kind": "norm", "dtype": dtype, "batch": b, "length": length, "dim": dim, "gate": gate,
                         "residual_scale": residual_scale, "rms": rms})


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = _TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=t):
        x = torch.empty(*shape, device="cuda", dtype=dtype)
        return x.normal_(0.0, scale, generator=g)

    def whole(low, high, *shape):
        return torch.randint(low, high, shape, device="cuda", generator=g)

    c = case
    s = {"case": dict(case)}
    if c["kind"] in ("attention", "prompt"):
        b, n, d = c["batch"], c["length"], c["head_dim"]
        s["q"] = normal(b, n, c["heads"], d, scale=1.5)
        s["k"], s["v"] = normal(b, n, c["kv_heads"], d, scale=1.5), normal(b, n, c["kv_heads"], d)
        if c["kind"] == "attention":
            s["dout"] = normal(b, n, c["heads"], d)
            s["valid"] = torch.arange(n, device="cuda") < whole(n // 2, n + 1, b, 1) if c["ragged"] else None
            for x in (s["q"], s["k"], s["v"]):
                x.requires_grad_()
        else:
            s["lengths"] = whole(min(n, max(1, n // 4)), n + 1, b)
            s["valid"] = torch.arange(n, device="cuda") < s["lengths"].unsqueeze(1)
            slots = c["sinks"] + c["window"]
            s["cache_k"] = torch.zeros(b, c["kv_heads"], slots, d, device="cuda", dtype=t)
            s["cache_v"] = torch.zeros_like(s["cache_k"])
    elif c["kind"] == "step":
        b, d, slots = c["batch"], c["head_dim"], c["sinks"] + c["window"]
        s["q"] = normal(b, c["heads"], d, scale=1.5)
        s["k"], s["v"] = normal(b, c["kv_heads"], d, scale=1.5), normal(b, c["kv_heads"], d)
        s["cache_k"] = normal(b, c["kv_heads"], slots, d, scale=1.5)
        s["cache_v"] = normal(b, c["kv_heads"], slots, d)
        s["lengths"] = whole(slots // 2, 3 * slots, b)  # tokens before this one: the ring partly or wholly filled
    elif c["kind"] == "distill":
        n, items, top = c["rows"], c["items"], c["top"]
        s["logits"] = normal(n, items, scale=2.0)
        ids = whole(0, items, n, top)
        near = s["logits"].gather(1, ids).float() + torch.empty(n, top, device="cuda").normal_(2.0, 1.0, generator=g)
        s["teacher_logits"], order = near.sort(1, descending=True)
        kept = torch.arange(top, device="cuda") < whole((top + 1) // 2, top + 1, n, 1)
        s["teacher_ids"] = torch.where(kept, ids.gather(1, order), -1)  # shorter lists end in -1
        s["logits"].requires_grad_()
    else:
        b, n, d = c["batch"], c["length"], c["dim"]
        s["res"], s["y"] = normal(b, n, d, scale=2.0), normal(b, n, d, scale=0.7)
        shape = {"channel": (d,), "sequence": (b, 1, d), "row": (b, n, d)}.get(c["gate"])
        s["gate"] = None if shape is None else normal(*shape, scale=0.5)
        f = torch.float32
        s["post_w"], s["pre_w"] = 1 + normal(d, scale=0.2, dtype=f), 1 + normal(d, scale=0.2, dtype=f)
        s["post_b"] = None if c["rms"] else normal(d, scale=0.2, dtype=f)
        s["pre_b"] = None if c["rms"] else normal(d, scale=0.2, dtype=f)
        s["ds"], s["dz"] = normal(b, n, d), normal(b, n, d)
        for x in _norm_leaves(s):
            x.requires_grad_()
    return s


def _norm_leaves(s):
    named = [s[k] for k in ("res", "y", "gate", "post_w", "post_b", "pre_w", "pre_b")]
    return [x for x in named if x is not None]


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    c = s["case"]
    if own:
        return _own(c, s)
    with torch.no_grad():
        return {"attention": _attention_plain, "prompt": _prompt_plain, "step": _step_plain,
                "distill": _distill_plain, "norm": _norm_plain}[c["kind"]](c, s)


def _own(c, s):
    ops = _ops()
    if c["kind"] == "attention":
        out = ops.window_attention(s["q"], s["k"], s["v"], c["window"], sinks=c["sinks"], causal=c["causal"],
                                   valid=s["valid"])
        return [out, *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])]
    if c["kind"] == "prompt":
        out = ops.window_attention(s["q"], s["k"], s["v"], c["window"], sinks=c["sinks"], valid=s["valid"])
        ops.window_cache_fill(s["cache_k"], s["cache_v"], s["k"], s["v"], s["lengths"], sinks=c["sinks"])
        return [out, s["cache_k"], s["cache_v"]]
    if c["kind"] == "step":
        out = ops.window_attention_step(s["q"], s["k"], s["v"], s["cache_k"], s["cache_v"], s["lengths"],
                                        sinks=c["sinks"])
        return [out, s["cache_k"], s["cache_v"]]
    if c["kind"] == "distill":
        loss = ops.distill_cross_entropy(s["logits"], s["teacher_ids"], s["teacher_logits"], c["temperature"])
        return [loss, *torch.autograd.grad(loss, (s["logits"],))]
    out, z = ops.gated_residual_norm(s["res"], s["y"], s["post_w"], s["post_b"], s["pre_w"], s["pre_b"],
                                     gate=s["gate"], residual_scale=c["residual_scale"], rms=c["rms"])
    return [out, z, *torch.autograd.grad((out, z), _norm_leaves(s), (s["ds"], s["dz"]))]


def _visible(c, n, valid):
    """(batch or 1, 1, n, n): which key (last) a query sees."""
    at = torch.arange(n, device="cuda")
    back = at.unsqueeze(1) - at
    if c.get("causal", True):
        seen = (back >= 0) & ((back < c["window"]) | (at < c["sinks"]))
    else:
        seen = (back.abs() < c["window"]) | (at < c["sinks"])
    seen = seen[None, None]
    return seen if valid is None else seen & valid[:, None, None, :] & valid[:, None, :, None]


def _heads_first(x, group=1):
    """(batch, n, heads, d) in 32 bits as (batch, heads * group, n, d)"""
    return x.detach().float().transpose(1, 2).repeat_interleave(group, 1).contiguous()


def _weights(q, k, seen):
    """softmax of the visible scores; a row that sees nothing has no weights"""
    score = torch.where(seen, q @ k.transpose(-1, -2).contiguous() * q.shape[-1] ** -0.5, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, 1.0, total)


def _attention_forward(c, s):
    group = c["heads"] // c["kv_heads"]
    q, k, v = _heads_first(s["q"]), _heads_first(s["k"], group), _heads_first(s["v"], group)
    p = _weights(q, k, _visible(c, c["length"], s["valid"]))
    return q, k, v, p, p @ v


def _attention_plain(c, s):
    q, k, v, p, out = _attention_forward(c, s)
    dout, group, t = _heads_first(s["dout"]), c["heads"] // c["kv_heads"], s["q"].dtype
    scale = q.shape[-1] ** -0.5
    dv = p.transpose(-1, -2).contiguous() @ dout
    dp = dout @ v.transpose(-1, -2).contiguous()
    ds = p * (dp - (dout * out).sum(-1, keepdim=True)) * scale
    dq = ds @ k
    dk = ds.transpose(-1, -2).contiguous() @ q
    shared = [x.unflatten(1, (-1, group)).sum(2) for x in (dk, dv)]
    return [x.transpose(1, 2).contiguous().to(t) for x in (out, dq, *shared)]


def _prompt_plain(c, s):
    out = _attention_forward(c, s)[-1]
    slots, sinks, window = s["cache_k"].shape[2], c["sinks"], c["window"]
    slot = torch.arange(slots, device="cuda")
    last = s["lengths"].unsqueeze(1) - 1
    # the last position of the prompt that falls on a slot: sinks keep theirs, the others come around
    turn = last - torch.remainder(last - slot, window)
    at = torch.where(slot < sinks, slot.expand_as(turn), turn)
    filled = (at <= last) & (at >= torch.where(slot < sinks, 0, sinks))
    rows = at.clamp(0, c["length"] - 1)[:, :, None, None].expand(-1, -1, c["kv_heads"], c["head_dim"])
    for cache, x in ((s["cache_k"], s["k"]), (s["cache_v"], s["v"])):
        cache.copy_(torch.where(filled[:, None, :, None], x.gather(1, rows).transpose(1, 2), cache))
    return [out.transpose(1, 2).contiguous().to(s["q"].dtype), s["cache_k"], s["cache_v"]]


def _step_plain(c, s):
    slots, sinks, n = s["cache_k"].shape[2], c["sinks"], s["lengths"]
    to = torch.where(n < sinks, n, sinks + torch.remainder(n - sinks, c["window"]))
    users = torch.arange(c["batch"], device="cuda")
    s["cache_k"][users, :, to] = s["k"]
    s["cache_v"][users, :, to] = s["v"]
    group = c["heads"] // c["kv_heads"]
    held = torch.arange(slots, device="cuda") < (n + 1).clamp(max=slots).unsqueeze(1)
    q = s["q"].float().unflatten(1, (c["kv_heads"], group))
    p = _weights(q, s["cache_k"].float(), held[:, None, None, :])
    out = p @ torch.where(held[:, None, :, None], s["cache_v"].float(), 0.0)
    return [out.flatten(1, 2).to(s["q"].dtype), s["cache_k"], s["cache_v"]]


def _distill_plain(c, s):
    x, ids, tau = s["logits"].detach().float() / c["temperature"], s["teacher_ids"], c["temperature"]
    there = ids >= 0
    t = torch.where(there, s["teacher_logits"].float() / tau, -math.inf)
    e = torch.exp(t - t.amax(1, keepdim=True))
    p = e / e.sum(1, keepdim=True)
    log_p = t - t.amax(1, keepdim=True) - e.sum(1, keepdim=True).log()
    top = x.amax(1, keepdim=True)
    ex = torch.exp(x - top)
    total = ex.sum(1, keepdim=True)
    log_q = x.gather(1, ids.clamp(min=0)) - top - total.log()
    rows = torch.where(there & (p > 0), p * (log_p - log_q), 0.0).sum(1)
    loss = tau * tau * rows.mean()
    grad = ex / total
    grad.scatter_add_(1, ids.clamp(min=0), torch.where(there, -p, 0.0))
    return [loss, (grad * (tau / c["rows"])).to(s["logits"].dtype)]


def _normed(x, rms):
    """the normalised rows and 1 / their deviation"""
    x = x if rms else x - x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-5)
    return x * r, r


def _norm_back(d, h, r, rms):
    """gradient of _normed's input for a gradient d of the normalised rows h"""
    d = d - h * (d * h).mean(-1, keepdim=True)
    return (d if rms else d - d.mean(-1, keepdim=True)) * r


def _norm_plain(c, s):
    t, rms = s["res"].dtype, c["rms"]
    f = {k: s[k].detach().float() for k in ("res", "y", "ds", "dz", "post_w", "pre_w")}
    post_b, pre_b = (0.0, 0.0) if rms else (s["post_b"].detach(), s["pre_b"].detach())
    gate = 1.0 if s["gate"] is None else s["gate"].detach().float()
    y, ry = _normed(f["y"], rms)
    branch = y * f["post_w"] + post_b
    out = c["residual_scale"] * f["res"] + gate * branch
    o, ro = _normed(out, rms)
    z = o * f["pre_w"] + pre_b
    d = f["ds"] + _norm_back(f["dz"] * f["pre_w"], o, ro, rms)
    db = d * gate
    dy = _norm_back(db * f["post_w"], y, ry, rms)
    grads = [(c["residual_scale"] * d).to(t), dy.to(t)]
    if c["gate"] != "none":
        over = {"channel": (0, 1), "sequence": (1,), "row": ()}[c["gate"]]
        dg = d * branch
        grads.append((dg.sum(over).reshape(s["gate"].shape) if over else dg).to(t))
    grads.append((db * y).sum((0, 1)))
    grads += [] if rms else [db.sum((0, 1))]
    grads.append((f["dz"] * o).sum((0, 1)))
    grads += [] if rms else [f["dz"].sum((0, 1))]
    return [out.to(t), z.to(t), *grads]


# ------------------------------------------------------------------------------------------------ what a pass needs
def _pairs(length, window, sinks, causal):
    """(query, key) pairs that a sequence of `length` tokens sees"""
    w = min(window, length)
    near = length * w - w * (w - 1) // 2
    # a sink that has left the window: for every query behind it
    far = sum(max(0, length - j - w) for j in range(min(sinks, length)))
    if causal:
        return near + far
    return 2 * near - length + far


def work(case):
    c = case
    size = 4 if c["dtype"] == "float32" else 2
    if c["kind"] in ("attention", "prompt"):
        q, kv = (c["batch"] * c["length"] * h * c["head_dim"] for h in (c["heads"], c["kv_heads"]))
        # ragged sequences hold three quarters (attention) or five eighths (prompt) of the padded length on average
        share = 0.75 if c.get("ragged") else 0.625 if c["kind"] == "prompt" else 1.0
        pairs = c["batch"] * c["heads"] * _pairs(max(1, int(c["length"] * share)), c["window"], c["sinks"],
                                                 c.get("causal", True))
        if c["kind"] == "prompt":
            cache = c["batch"] * c["kv_heads"] * c["head_dim"] * min(c["length"], c["window"] + c["sinks"])
            return {"bytes": int(size * share * (2 * q + 2 * kv) + 2 * size * cache), "flops": 4 * pairs * c["head_dim"]}
        # two products forward; the scores again, the weights' gradient and those of q, k, v backward
        return {"bytes": int(size * (2 * q + 2 * kv + share * (2 * q + 2 * kv) + q)),
                "flops": 14 * pairs * c["head_dim"]}
    if c["kind"] == "step":
        slots = c["sinks"] + c["window"]
        held = c["batch"] * slots * 0.95
        new = c["batch"] * (2 * c["heads"] + 4 * c["kv_heads"]) * c["head_dim"]
        return {"bytes": int(size * (2 * held * c["kv_heads"] * c["head_dim"] + new)),
                "flops": int(4 * held * c["heads"] * c["head_dim"])}
    if c["kind"] == "distill":
        n = c["rows"] * c["items"]
        return {"bytes": 2 * size * n + 12 * c["rows"] * c["top"], "flops": 8 * n}
    n = c["batch"] * c["length"] * c["dim"]
    gates = {"none": 0, "channel": c["dim"], "sequence": c["batch"] * c["dim"], "row": n}[c["gate"]]
    # in: res, y and the two outputs' gradients; out: the two outputs and the gradients of res and y
    return {"bytes": size * (8 * n + 2 * gates) + 4 * 8 * c["dim"], "flops": 40 * n}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    c = case
    s = prepare(case, seed)
    big = {k: v.detach().double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in s.items()}
    if c["kind"] in ("attention", "prompt"):
        return _exact_attention(c, s, big)
    if c["kind"] == "step":
        return _exact_step(c, s, big)
    if c["kind"] == "distill":
        return _exact_distill(c, big)
    return _exact_norm(c, big)


def _exact_attention(c, s, big):
    """one key head of one sequence at a time, its weights by log-sum-exp, its gradients by autograd"""
    b, n, kv = c["batch"], c["length"], c["kv_heads"]
    group, causal = c["heads"] // kv, c.get("causal", True)
    if b * c["heads"] * n * n * c["head_dim"] > 2 ** 43 or b * kv > 4096:
        return None
    grads = c["kind"] == "attention"
    i = torch.arange(n, device="cuda").view(-1, 1)
    j = i.view(1, -1)
    near = ((i - j < c["window"]) & (j <= i)) if causal else ((i - j < c["window"]) & (j - i < c["window"]))
    seen = near | ((j < c["sinks"]) & ((j <= i) if causal else (j >= 0)))
    out, dq = torch.zeros_like(big["q"]), torch.zeros_like(big["q"])
    dk, dv = torch.zeros_like(big["k"]), torch.zeros_like(big["k"])
    for u in range(b):
        m = n if s["valid"] is None else int(s["valid"][u].sum())
        if m == 0:
            continue
        hidden = ~seen[:m, :m].unsqueeze(0)
        for h in range(kv):
            of = slice(h * group, (h + 1) * group)
            q = big["q"][u, :m, of].permute(1, 0, 2).clone().requires_grad_(grads)
            k = big["k"][u, :m, h].clone().requires_grad_(grads)
            v = big["v"][u, :m, h].clone().requires_grad_(grads)
            score = (torch.matmul(q, k.t()) / math.sqrt(c["head_dim"])).masked_fill(hidden, -math.inf)
            o = torch.matmul((score - torch.logsumexp(score, -1, keepdim=True)).exp(), v)
            out[u, :m, of] = o.detach().permute(1, 0, 2)
            if grads:
                a, e, f = torch.autograd.grad(o, (q, k, v), big["dout"][u, :m, of].permute(1, 0, 2))
                dq[u, :m, of], dk[u, :m, h], dv[u, :m, h] = a.permute(1, 0, 2), e, f
    if grads:
        return [out, dq, dk, dv]
    caches = []
    for x, cache in ((big["k"], big["cache_k"]), (big["v"], big["cache_v"])):
        for u, m in enumerate(s["lengths"].tolist()):
            kept = min(m, c["sinks"])
            cache[u, :, :kept] = x[u, :kept].transpose(0, 1)
            late = torch.arange(max(c["sinks"], m - c["window"]), max(c["sinks"], m), device="cuda")
            cache[u, :, c["sinks"] + (late - c["sinks"]) % c["window"]] = x[u, late].transpose(0, 1)
        caches.append(cache)
    return [out, *caches]


def _exact_step(c, s, big):
    group, out = c["heads"] // c["kv_heads"], torch.zeros_like(big["q"])
    for u, m in enumerate(s["lengths"].tolist()):
        to = m if m < c["sinks"] else c["sinks"] + (m - c["sinks"]) % c["window"]
        held = min(m + 1, c["sinks"] + c["window"])
        big["cache_k"][u, :, to], big["cache_v"][u, :, to] = big["k"][u], big["v"][u]
        k, v = big["cache_k"][u, :, :held], big["cache_v"][u, :, :held]
        q = big["q"][u].view(c["kv_heads"], group, c["head_dim"])
        score = torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(c["head_dim"])
        out[u] = torch.matmul(torch.softmax(score, -1), v).view(c["heads"], c["head_dim"])
    return [out, big["cache_k"], big["cache_v"]]


def _exact_distill(c, big):
    """the loss by log-softmax and its gradient by autograd, some rows at a time"""
    tau, total, grads = c["temperature"], 0.0, []
    for x, ids, teacher in zip(big["logits"].split(256), big["teacher_ids"].split(256),
                               big["teacher_logits"].split(256)):
        x = x.clone().requires_grad_()
        absent = ids < 0
        log_p = torch.log_softmax((teacher / tau).masked_fill(absent, -math.inf), 1)
        log_q = torch.log_softmax(x / tau, 1).gather(1, ids.masked_fill(absent, 0))
        part = (log_p.exp() * (log_p.masked_fill(absent, 0.0) - log_q)).sum() * (tau * tau / c["rows"])
        grads.append(torch.autograd.grad(part, x)[0])
        total = total + part.detach()
    return [total, torch.cat(grads)]


def _exact_norm(c, big):
    """as functions of the definition, gradients by autograd"""
    leaves = [x.requires_grad_() for x in _norm_leaves(big)]

    def norm(x, w, b):
        if not c["rms"]:
            x = x - x.mean(-1, keepdim=True)
        x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-5) * w
        return x if b is None else x + b

    branch = norm(big["y"], big["post_w"], big["post_b"])
    out = c["residual_scale"] * big["res"] + (branch if big["gate"] is None else big["gate"] * branch)
    z = norm(out, big["pre_w"], big["pre_b"])
    return [out.detach(), z.detach(), *torch.autograd.grad((out, z), leaves, (big["ds"], big["dz"]))]
