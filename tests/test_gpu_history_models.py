"""GPU: the long-history operators as the models, training modules and serving calls use them."""
import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
V, L, D, H = 60, 24, 64, 2
BASE = dict(transformer_hidden_size=D, num_transformer_heads=H, num_transformer_layers=2, item_vocab_size=V,
            max_seq_length=L, transformer_dropout=0.0)


def model(asme, cls="SASRecModel", seed=0, **how):
    torch.manual_seed(seed)
    return getattr(asme, cls)(**{**BASE, **how}).cuda()


def histories(asme, b, n, seed, shortest=1):
    g = torch.Generator().manual_seed(seed)
    lengths = torch.randint(shortest, n + 1, (b,), generator=g)
    lengths[0] = n
    items = torch.randint(3, V, (b, n), generator=g)
    mask = torch.arange(n) < lengths[:, None]
    items = torch.where(mask, items, 0).cuda()
    return asme.InputSequence(items, mask.cuda()), lengths


def test_a_window_over_everything_is_full_attention(asme, dev):
    full, wide = model(asme), model(asme, attention_window=L)
    wide.load_state_dict(full.state_dict())
    seq, lengths = histories(asme, 5, L, 1)
    with torch.no_grad():
        a, b = full.eval().encode(seq), wide.eval().encode(seq)
    on = seq.padding_mask
    # two fp32 kernels for the same sums, through two blocks: a few hundred roundings of O(1) terms
    assert (a[on] - b[on]).abs().max() < 2e-5 * a[on].abs().max()


def reference_layer(layer, x, key_valid, causal, window, sinks):
    """the gated blocks by torch in 64 bits, from the layer's own parameters"""
    p = {k: v.detach().double().requires_grad_() for k, v in layer.named_parameters()}
    x = x.detach().double().requires_grad_()
    n = x.shape[1]
    i, j = torch.arange(n, device=x.device)[:, None], torch.arange(n, device=x.device)[None]
    seen = ((i - j < window) | (j < sinks)) & (j <= i) if causal else ((i - j).abs() < window) | (j < sinks)
    seen = seen & key_valid[:, None, None, :] & key_valid[:, None, :, None]

    def norm(h, name):
        return F.layer_norm(h, (D,), p[name + ".weight"], p[name + ".bias"], 1e-5)

    h = x
    for k in range(len(layer.transformer_blocks)):
        b = f"transformer_blocks.{k}."
        z = norm(h, b + "input_sublayer.norm")
        q, kk, v = (F.linear(z, p[f"{b}attention.linear_layers.{u}.weight"], p[f"{b}attention.linear_layers.{u}.bias"])
                    .view(*z.shape[:2], H, D // H).transpose(1, 2) for u in range(3))
        s = (q @ kk.transpose(-1, -2).contiguous() / math.sqrt(D // H)).masked_fill(~seen, -math.inf)
        o = (torch.softmax(s, -1).nan_to_num(0.0) @ v).transpose(1, 2).reshape(z.shape)
        a = F.linear(o, p[b + "attention.output_linear.weight"], p[b + "attention.output_linear.bias"])
        h = h + p[b + "input_gate.gate"] * norm(a, b + "input_gate.norm")
        z = norm(h, b + "output_sublayer.norm")
        f = F.gelu(F.linear(z, p[b + "feed_forward.w_1.weight"], p[b + "feed_forward.w_1.bias"]))
        f = F.linear(f, p[b + "feed_forward.w_2.weight"], p[b + "feed_forward.w_2.bias"])
        h = h + p[b + "output_gate.gate"] * norm(f, b + "output_gate.norm")
    return x, p, h


@pytest.mark.parametrize("causal", [True, False])
def test_gated_blocks_and_their_gradients(asme, dev, causal):
    torch.manual_seed(3)
    layer = asme.layers.TransformerLayer(D, H, 2, 4 * D, 0.0, attention_window=5, attention_sinks=2,
                                         gated_norms=True).cuda()
    with torch.no_grad():
        for name, p in layer.named_parameters():
            if "gate" in name or "norm" in name:
                p.add_(0.2 * torch.randn_like(p))
    x = torch.randn(3, L, D, device=dev, requires_grad=True)
    valid = torch.arange(L, device=dev) < torch.tensor([[L], [7], [1]], device=dev)
    out = layer(x, asme.layers.key_valid_mask(valid, x.shape), causal)
    w = torch.randn_like(out) * valid[..., None]  # (what padding comes to is no one's)
    x64, p64, want = reference_layer(layer, x, valid, causal, 5, 2)
    assert (out[valid] - want[valid]).abs().max() < 1e-5 * want[valid].abs().max()
    names = [n for n, _ in layer.named_parameters()]
    got = torch.autograd.grad(out, [x, *layer.parameters()], w)
    ref = torch.autograd.grad(want, [x64, *p64.values()], w.double())
    size = {n: b.abs().max() for n, b in zip(["x", *names], ref)}
    for n, a, b in zip(["x", *names], got, ref):
        # sums over 32 rows and 256 columns of fp32 products, each a few hundred roundings: 2^-24 * 300 of the largest.
        # The keys' bias alone has none that is large: a softmax does not change when every score of a row gains q . b,
        # so its gradient sum_ij dS_ij q_i is 0 (sum_j dS_ij = 0), and what fp32 leaves of it is the roundings of terms
        # that are as large as those of the keys' weights, sum_ij dS_ij q_i z_j with |z| ~ 1
        terms = size[n.replace("bias", "weight")] if n.endswith("linear_layers.1.bias") else size[n]
        assert (a - b).abs().max() < 5e-5 * terms.clamp(min=1e-3), n


@pytest.mark.parametrize("window,sinks,gated", [(4, 0, False), (5, 2, True), (L, 1, False)])
def test_decode_gives_what_the_whole_history_gives(asme, dev, window, sinks, gated):
    m = model(asme, attention_window=window, attention_sinks=sinks, gated_norms=gated).eval()
    n, steps = 9, 12
    seq, lengths = histories(asme, 4, n, 5)
    g = torch.Generator().manual_seed(6)
    extra = torch.randint(3, V, (steps, 4), generator=g).cuda()
    rep, caches = m.prefill(seq)
    whole = torch.zeros(4, L, dtype=torch.int64, device=dev)
    whole[:, :n] = seq.sequence
    for t in range(steps + 1):
        now = lengths + t
        mask = (torch.arange(L) < now[:, None]).cuda()
        with torch.no_grad():
            want = m.encode(asme.InputSequence(whole, mask))[torch.arange(4), now.cuda() - 1]
        assert (rep - want).abs().max() < 2e-5 * want.abs().max(), t
        assert torch.equal(caches.lengths.cpu(), now)
        if t < steps:
            whole[torch.arange(4), now.cuda()] = extra[t]
            rep = m.decode(extra[t], caches)
    top = asme.ops.catalog_topk(rep, m.item_table().detach(), 5)
    score = rep.double() @ m.item_table().detach().double().t()
    assert torch.equal(top[1].sort(1).values, score.topk(5).indices.sort(1).values)
    while caches.most < L:
        m.decode(extra[0], caches)
    with pytest.raises(IndexError, match="max_seq_len"):
        m.decode(extra[0], caches)
    with pytest.raises(ValueError, match="one for each"):
        m.decode(extra[0][:2], caches)


def test_prompts_padded_to_the_models_length(asme, dev):
    """how far decode() goes is the longest history's matter, not its padding's; padding in front is refused"""
    m = model(asme, attention_window=5, attention_sinks=1).eval()
    seq, lengths = histories(asme, 4, 9, 5)
    whole = torch.zeros(4, L, dtype=torch.int64, device=dev)
    whole[:, :9] = seq.sequence
    mask = (torch.arange(L) < lengths[:, None]).cuda()
    item = torch.full((4,), 3, dtype=torch.int64, device=dev)
    want = m.decode(item, m.prefill(seq)[1])
    rep, caches = m.prefill(asme.InputSequence(whole, mask))
    assert caches.most == int(lengths.max()) < L
    assert torch.equal(m.decode(item, caches), want)
    with pytest.raises(ValueError, match="right-padded"):
        m.prefill(asme.InputSequence(whole.flip(1), mask.flip(1)))


def cloze_batch(asme, b, seed, users=False):
    seq, lengths = histories(asme, b, L, seed, shortest=4)
    g = torch.Generator().manual_seed(seed + 1)
    hidden = (torch.rand(b, L, generator=g) < 0.3).cuda() & seq.padding_mask
    hidden[:, 0] = True
    batch = {"item": seq.sequence.masked_fill(hidden, 1), "item.target": seq.sequence.masked_fill(~hidden, 0)}
    batch["teacher.ids"] = torch.randint(-1, V, (b, L, 7), generator=g).cuda()
    batch["teacher.logits"] = torch.randn(b, L, 7, generator=g).cuda()
    if users:
        batch["gender"] = torch.randint(0, 3, (b, L, 1), generator=g).cuda()
    return batch


def mixed64(logits, targets, ids, t, weight, tau):
    x = logits.double()
    there = ids >= 0
    p = torch.softmax((t.double() / tau).masked_fill(~there, -math.inf), 1).nan_to_num(0.0)
    q = torch.log_softmax(x / tau, 1).gather(1, ids.clamp(min=0))
    kd = torch.where(p > 0, p * (p.clamp(min=1e-300).log() - q), 0.0).sum() * tau * tau / there.any(1).sum()
    return weight * kd + (1 - weight) * F.cross_entropy(x, targets)


@pytest.mark.parametrize("cls,module", [("BERT4RecModel", "MaskedTrainingModule"),
                                        ("SASRecModel", "NextItemPredictionTrainingModule")])
def test_training_on_a_teachers_lists(asme, dev, cls, module):
    how = {"mode": "full"} if cls == "SASRecModel" else {}
    m = model(asme, cls, attention_window=6, attention_sinks=1, gated_norms=True, **how)
    train = getattr(asme, module)(model=m, item_tokenizer=asme.tokenization.Tokenizer(V - 3), metrics=None)
    train.distillation = asme.losses.TopKDistillationLoss(temperature=2.0, weight=0.3)
    batch = cloze_batch(asme, 6, 11)
    with pytest.raises(Exception, match="teacher"):
        train.training_step({k: v for k, v in batch.items() if "teacher" not in k}, 0)
    with pytest.raises(ValueError, match="targets"):
        train.training_step({**batch, "teacher.ids": batch["teacher.ids"][:, 1:]}, 0)
    train.train()
    opt = train.configure_optimizers()
    opt = asme.modules.split_optimizers(opt)[0]
    opt.zero_grad()
    loss = train.training_step(batch, 0)["loss"]
    rows = batch["item.target"].reshape(-1).nonzero().squeeze(1)
    with torch.no_grad():
        logits = m.forward_rows(asme.InputSequence(batch["item"], batch["item"].ne(0)), rows)
    want = mixed64(logits, batch["item.target"].reshape(-1)[rows], batch["teacher.ids"].reshape(-1, 7)[rows],
                   batch["teacher.logits"].reshape(-1, 7)[rows], 0.3, 2.0)
    # two losses of O(1) .. O(10) from the same fp32 logits
    assert abs(loss.item() - want.item()) < 1e-5 * abs(want.item())
    loss.backward()
    # (the masked module's warm-up starts from a learning rate of 0: gradients, not steps, show what is reached)
    reached = [n for n, p in m.named_parameters() if p.grad is not None and p.grad.abs().sum() > 0]
    assert any("gate" in n for n in reached) and any("linear_layers" in n for n in reached) and len(reached) > 20
    opt.step()
    m.flush_table()
    assert all(torch.isfinite(p).all() for p in m.parameters())


def test_distillation_with_a_user_token(asme, dev):
    tok = {"tokenizers.gender": range(3)}
    torch.manual_seed(0)
    m = asme.UBERT4RecModel(**BASE, additional_attributes=None, additional_tokenizers=tok,
                            user_attributes={"gender": {"embedding_type": "user_embedding"}}, positional_embedding=True,
                            segment_embedding=True, attention_window=5, attention_sinks=1).cuda()
    train = asme.UBERTMaskedTrainingModule(model=m, item_tokenizer=asme.tokenization.Tokenizer(V - 3), metrics=None)
    train.distillation = asme.losses.TopKDistillationLoss(temperature=1.0, weight=0.5)
    batch = cloze_batch(asme, 4, 21, users=True)
    batch["gender"] = batch["gender"].squeeze(-1)
    loss = train.training_step(dict(batch), 0)["loss"]
    rows = F.pad(batch["item.target"], (1, 0)).reshape(-1).nonzero().squeeze(1)
    items = batch["item.target"].reshape(-1).nonzero().squeeze(1)
    with torch.no_grad():
        seq = asme.InputSequence(batch["item"], batch["item"].ne(0), {"gender": batch["gender"]})
        logits = m.forward_rows(seq, rows)
    want = mixed64(logits, batch["item.target"].reshape(-1)[items], batch["teacher.ids"].reshape(-1, 7)[items],
                   batch["teacher.logits"].reshape(-1, 7)[items], 0.5, 1.0)
    assert abs(loss.item() - want.item()) < 1e-5 * abs(want.item())
    loss.backward()
    # the user's row reaches far positions through the sink: its embedding has a gradient
    grads = {n: p.grad for n, p in m.named_parameters() if "user_attribute" in n}
    assert grads and all(g.abs().sum() > 0 for g in grads.values())


def test_a_student_from_teacher_to_server(asme, dev):
    """a teacher's best items teach a windowed, gated student, which then serves growing histories"""
    teacher = model(asme, seed=1, mode="full").eval()
    student = model(asme, seed=2, mode="full", attention_window=6, attention_sinks=1, gated_norms=True)
    train = asme.NextItemPredictionTrainingModule(model=student, item_tokenizer=asme.tokenization.Tokenizer(V - 3),
                                                  metrics=None)
    train.distillation = asme.losses.TopKDistillationLoss(temperature=1.5, weight=0.8)
    opt = asme.modules.split_optimizers(train.configure_optimizers())[0]
    for step in range(3):
        batch = cloze_batch(asme, 6, 31 + step)
        with torch.no_grad():
            h = teacher.encode(asme.InputSequence(batch["item"], batch["item"].ne(0)))
            w, b = teacher.head_weight_bias()
            val, idx = asme.ops.catalog_topk(h.view(-1, D), w.detach(), 8, b.detach())
        batch["teacher.ids"], batch["teacher.logits"] = idx.view(6, L, 8), val.view(6, L, 8)
        opt.zero_grad()
        loss = train.training_step(batch, step)["loss"]
        loss.backward()
        opt.step()
        assert torch.isfinite(loss)
    student.eval().flush_table()
    seq, lengths = histories(asme, 5, 10, 41)
    rep, caches = student.prefill(seq)
    w, b = (t.detach() for t in student.head_weight_bias())
    for _ in range(6):
        val, idx = asme.ops.catalog_topk(rep, w, 3, b)
        want = (rep.double() @ w.double().t() + b.double()).topk(3)
        assert (val - want.values).abs().max() < 1e-5 * want.values.abs().max()
        rep = student.decode(idx[:, 0].contiguous(), caches)
    assert torch.equal(caches.lengths.cpu(), lengths + 6)
