"""GPU: the tuning operators together, on a context's model: log-probabilities of a batch,
a preference or policy loss on them, the backward to the adapters and a Muon step, against
the CPU oracle's model with float64 losses; and through the reference-compatible API's logits.

Bars: the step's own, a loss within 1e-3 and every adapter gradient within 1e-2 relative
L2 of the fp32 oracle."""
import copy
import ctypes as C

import pytest
import torch
import torch.nn.functional as F

import llmt
from helpers import SMALL, grad_errors, rel_l2, small_problem, upload_model
from oracle import lora_step as ref
from oracle.configs import quantize_model_int8

pytestmark = pytest.mark.gpu


def context(dev, W, ad, batch, seq_len):
    ctx = llmt.Context(llmt.make_dims(SMALL), max_batch=batch, seq_len=seq_len)
    upload_model(ctx, W, dev)
    ctx.lora_set("param", llmt.flatten_adapters(ad).to(dev))
    return ctx


def prompts_out(tgt, seed=0):
    """Targets without a random prompt of each window and its last position."""
    g = torch.Generator().manual_seed(seed)
    t = tgt.clone()
    t[:, -1] = -1
    for b in range(t.shape[0]):
        t[b, :int(torch.randint(0, t.shape[1] // 2, (1,), generator=g))] = -1
    return t


def oracle_logp(logits, tgt):
    """logp [T] in float64 with autograd, 0 without a target."""
    t = tgt.reshape(-1).long()
    lp = torch.log_softmax(logits.double(), 1).gather(1, t.clamp(min=0)[:, None])[:, 0]
    return torch.where(t >= 0, lp, torch.zeros_like(lp))


def oracle_grads(W, ad, tok, tgt, loss_of):
    """Loss and adapter gradients of loss_of(logp) through the oracle's model."""
    B, S = tok.shape
    logits, stash = ref.model_forward(W, ad, tok, SMALL)
    x = logits.detach().double().requires_grad_()
    loss = loss_of(oracle_logp(x, tgt))
    loss.backward()
    grads, _ = ref.model_backward(x.grad.float(), stash, W, ad, SMALL, B, S, ())
    return float(loss.detach()), grads


@pytest.mark.parametrize("batch,seq_len", [(2, 64), (3, 37), (1, 2)])
def test_context_logprobs(dev, batch, seq_len):
    W, ad, tok, tgt = small_problem(batch=batch, seq_len=seq_len)
    tgt = prompts_out(tgt)
    ctx = context(dev, W, ad, batch, seq_len)
    try:
        lp = ctx.forward_logprobs(tok.to(dev), tgt.to(dev))
        n = batch * seq_len
        logits = ctx.logits(n)
        # the same logits through the standalone operator: both sum V / 64 terms a lane or
        # fewer, 2^-24 each, and round logarithms and differences once
        alone, _, _ = llmt.token_logprobs(logits, tgt.reshape(-1).to(dev))
        tol = (SMALL.vocab / 64 + 60) * 2.0 ** -24
        assert ((lp - alone).abs() <= tol + 2.0 ** -22 * alone.abs()).all()
        assert (lp.cpu()[tgt.reshape(-1) < 0] == 0).all()
        want = oracle_logp(ref.model_forward(W, ad, tok, SMALL)[0], tgt)
        count = max(1, int((tgt >= 0).sum()))
        assert abs(float(lp.sum()) - float(want.sum())) / count < 1e-3
    finally:
        ctx.close()


@pytest.mark.parametrize("batch,seq_len", [(2, 64), (3, 37)])
def test_context_backward_of_any_function(dev, batch, seq_len):
    """Random weights on the log-probabilities, some 0 and of either sign."""
    W, ad, tok, tgt = small_problem(batch=batch, seq_len=seq_len)
    tgt = prompts_out(tgt, 1)
    g = torch.Generator().manual_seed(3)
    w = torch.randn(batch * seq_len, generator=g)
    w[torch.rand(batch * seq_len, generator=g) < 0.3] = 0.0
    _, grads = oracle_grads(W, ad, tok, tgt, lambda lp: (w.double() * lp).sum())
    ctx = context(dev, W, ad, batch, seq_len)
    try:
        ctx.forward_logprobs(tok.to(dev), tgt.to(dev))
        for _ in range(2):  # again from the same stashes
            ctx.backward_logprobs(w.to(dev))
            errs = grad_errors(ctx.lora_get("grad"), grads, SMALL)
            assert max(errs.values()) < 1e-2, errs
    finally:
        ctx.close()


@pytest.mark.parametrize("weights", ["f16", "i8", "untied"])
def test_context_backward_equals_the_cross_entropy_step(dev, weights):
    """dlogp = -1 / n on the rows with a target is the mean cross entropy: the same gradient
    as llmt_forward_backward up to fp16 roundings that fall to the other side.  Where the two
    sides' values differ by a relative d, one in d / 2^-10 rounds to another neighbour, a step
    of at most 2^-10 away: each rounding adds at most d 2^-10 to the mean square d^2, so d
    grows by 2^-11 a rounding.  There are 16 on the longest path of two layers (the head's
    operand and the final norm's; per layer the SwiGLU's, both norms', dO, P, dS and the
    Q/K/V operand), and the fp32 differences before them are 1e-6: 16 x 2^-11."""
    W, ad, tok, tgt = small_problem()
    B, S = tok.shape
    if weights == "i8":
        W, qs = quantize_model_int8(copy.deepcopy(W))
        ctx = llmt.Context(llmt.make_dims(SMALL), B, S, int8=True)
        f = lambda t: t.float().to(dev).contiguous()
        for l, lw in enumerate(W.layers):
            q = [qs[(l, n)] for n in ("wq", "wk", "wv", "wo", "w_gate", "w_up", "w_down")]
            ctx.set_layer_i8(l, [torch.from_numpy(a).to(dev) for a, _ in q],
                             [torch.from_numpy(b).to(dev) for _, b in q], f(lw.attn_norm),
                             f(lw.ffn_norm), f(lw.q_norm), f(lw.k_norm))
        ctx.set_embed_f16(W.embed.half().to(dev), f(W.final_norm))
        ctx.lora_set("param", llmt.flatten_adapters(ad).to(dev))
    else:
        ctx = context(dev, W, ad, B, S)
    if weights == "untied":
        g = torch.Generator().manual_seed(4)
        ctx.set_lm_head_f16((torch.randn(SMALL.vocab, SMALL.hidden, generator=g) * 0.02).half().to(dev))
    try:
        loss = ctx.forward_backward(tok.to(dev), tgt.to(dev))
        want = ctx.lora_get("grad")
        t = tgt.clone()
        t[:, -1] = -1
        lp = ctx.forward_logprobs(tok.to(dev), t.to(dev))
        n = B * (S - 1)
        assert abs(loss + float(lp.double().sum()) / n) < 1e-5
        d = torch.where(t.reshape(-1) >= 0, -1.0 / n, 0.0).to(dev)
        ctx.backward_logprobs(d)
        assert rel_l2(ctx.lora_get("grad"), want) < 16 * 2.0 ** -11
    finally:
        ctx.close()


def test_context_order_of_calls(dev):
    W, ad, tok, tgt = small_problem()
    B, S = tok.shape
    ctx = context(dev, W, ad, B, S)
    tok, tgt = tok.to(dev), tgt.to(dev)
    d = torch.zeros(B * S, device=dev)
    L = llmt.lib()
    try:
        assert L.llmt_backward_logprobs(ctx.h, llmt.ptr(d)) == llmt.LLMT_ERR_STATE
        x = torch.randn(B * S, SMALL.hidden, device=dev)
        for graph in (False, True):
            ctx.set_graph(graph)
            for other in (lambda: ctx.forward_backward(tok, tgt),
                          lambda: ctx.step(tok, tgt, llmt.hparams(), 1),
                          lambda: ctx.layer_forward(0, x, B),
                          lambda: ctx.layer_backward(0, x, B),
                          lambda: ctx.head_ce(x.half(), tgt.reshape(-1))):
                ctx.forward_logprobs(tok, tgt)
                ctx.backward_logprobs(d)
                other()
                assert L.llmt_backward_logprobs(ctx.h, llmt.ptr(d)) == llmt.LLMT_ERR_STATE
                assert "forward_logprobs" in L.llmt_last_error().decode()
        ctx.forward_logprobs(tok[:1], tgt[:1])
        with pytest.raises(llmt.LlmtError):
            ctx.backward_logprobs(d)               # another batch
        with pytest.raises(llmt.LlmtError):
            ctx.backward_logprobs(d[:S].double())
        assert L.llmt_backward_logprobs(ctx.h, None) == llmt.LLMT_ERR_ARG
        assert L.llmt_forward_logprobs(ctx.h, llmt.ptr(tok), llmt.ptr(tgt), B, None) == llmt.LLMT_ERR_ARG
        assert L.llmt_forward_logprobs(ctx.h, llmt.ptr(tok), llmt.ptr(tgt), B + 1, llmt.ptr(d)) == llmt.LLMT_ERR_ARG
    finally:
        ctx.close()


def test_context_refuses_a_backward_through_other_weights(dev):
    """Weights or adapters that changed after the forward are not those of its stashes."""
    W, ad, tok, tgt = small_problem()
    B, S = tok.shape
    ctx = context(dev, W, ad, B, S)
    tok, tgt = tok.to(dev), tgt.to(dev)
    d = torch.zeros(B * S, device=dev)
    L = llmt.lib()
    emb, norm = W.embed.half().to(dev), W.final_norm.float().to(dev)
    try:
        for other in (lambda: llmt.check(L.llmt_adamw(ctx.h, C.byref(llmt.hparams()), 1)),
                      lambda: ctx.muon(llmt.muon_hparams()),
                      lambda: ctx.lora_set("param", llmt.flatten_adapters(ad).to(dev)),
                      lambda: llmt.check(L.llmt_lora_init(ctx.h, 1, 0.02, 0.0)),
                      lambda: ctx.set_embed_f16(emb, norm),
                      lambda: ctx.set_lm_head_f16(emb)):
            ctx.forward_logprobs(tok, tgt)
            ctx.backward_logprobs(d)
            ctx.lora_set("grad", ctx.lora_get("grad"))
            ctx.backward_logprobs(d)
            other()
            assert L.llmt_backward_logprobs(ctx.h, llmt.ptr(d)) == llmt.LLMT_ERR_STATE
    finally:
        ctx.close()


def test_preference_step(dev):
    """Two pairs of answers: the reference's log-probabilities with the adapters off, the
    policy's with them on, the loss, the backward and two Muon steps."""
    B, S = 4, 48
    W, ad, tok, tgt = small_problem(batch=B, seq_len=S, seed=11)
    tgt = prompts_out(tgt, 2)
    off_ad = [{p: ref.Adapter(a.A, torch.zeros_like(a.B)) for p, a in d.items()} for d in ad]
    base = oracle_logp(ref.model_forward(W, off_ad, tok, SMALL)[0], tgt)
    beta = float(torch.tensor(0.5))

    def loss_of(lp):
        r = beta * (lp - base).view(B, S).sum(1)
        return F.softplus(-(r[0::2] - r[1::2])).mean()

    want, grads = oracle_grads(W, ad, tok, tgt, loss_of)
    ctx = context(dev, W, off_ad, B, S)
    tok, tgt = tok.to(dev), tgt.to(dev)
    offsets = torch.arange(0, B * S + 1, S, dtype=torch.int32, device=dev)
    try:
        ref_lp = ctx.forward_logprobs(tok, tgt)
        ctx.lora_set("param", llmt.flatten_adapters(ad).to(dev))
        hp = llmt.muon_hparams(lr=1e-3)
        p0, m0 = ctx.lora_get("param"), ctx.lora_get("m")
        for step in range(2):
            lp = ctx.forward_logprobs(tok, tgt)
            mean, losses, rewards, d = llmt.preference_loss(
                lp, ref_lp, offsets, beta=beta, mask=tgt.reshape(-1) >= 0)
            ctx.backward_logprobs(d)
            if step == 0:
                assert abs(float(mean) - want) < 1e-3
                errs = grad_errors(ctx.lora_get("grad"), grads, SMALL)
                assert max(errs.values()) < 1e-2, errs
            g = ctx.lora_get("grad")
            ctx.muon(hp)
            r, h, q, kv = 16, SMALL.hidden, SMALL.q_dim, SMALL.kv_dim
            llmt.muon_update(p0, g, m0, [(r, h), (q, r), (r, h), (kv, r), (r, h), (kv, r), (r, q),
                                         (h, r)], hp)
            assert torch.equal(ctx.lora_get("param"), p0)
    finally:
        ctx.close()


def test_policy_step(dev):
    """Sampled answers with an advantage each: the clipped loss with a KL term and an entropy
    bonus taken on the context's logits, and AdamW."""
    B, S = 3, 40
    W, ad, tok, tgt = small_problem(batch=B, seq_len=S, seed=12)
    tgt = prompts_out(tgt, 4)
    g = torch.Generator().manual_seed(1)
    base = oracle_logp(ref.model_forward(W, ad, tok, SMALL)[0], tgt)
    old = (base + 0.3 * torch.randn(B * S, generator=g)).float()
    refl = (base + 0.3 * torch.randn(B * S, generator=g)).float()
    adv = torch.tensor([1.0, -0.7, 0.4])
    keep = (tgt.reshape(-1) >= 0)

    def loss_of(lp):
        ratio = (lp - old.double()).exp()
        A = adv.double().repeat_interleave(S)
        pg = -torch.minimum(ratio * A, ratio.clamp(0.8, 1.2) * A)
        d = refl.double() - lp
        return ((pg + 0.1 * (d.exp() - d - 1)) * keep).sum() / keep.sum()

    want, grads = oracle_grads(W, ad, tok, tgt, loss_of)
    ctx = context(dev, W, ad, B, S)
    tok, tgt = tok.to(dev), tgt.to(dev)
    offsets = torch.arange(0, B * S + 1, S, dtype=torch.int32, device=dev)
    try:
        lp = ctx.forward_logprobs(tok, tgt)
        p = llmt.policy_loss(lp, old.to(dev), adv.to(dev), offsets, ref_logp=refl.to(dev),
                             mask=keep.to(dev), kl_coef=0.1, per_sequence=True)
        assert abs(float(p.loss) - want) < 1e-3
        ctx.backward_logprobs(p.dlogp)
        errs = grad_errors(ctx.lora_get("grad"), grads, SMALL)
        assert max(errs.values()) < 1e-2, errs
        before = ctx.lora_get("param")
        check = llmt.lib().llmt_adamw(ctx.h, C.byref(llmt.hparams()), 1)
        assert check == 0 and not torch.equal(ctx.lora_get("param"), before)
        # the same gradients by way of the logits, with the entropy's share on top
        logits = ctx.logits(B * S)
        lp2, st, ent = llmt.token_logprobs(logits, tgt.reshape(-1), want_entropy=True)
        p2 = llmt.policy_loss(lp2, old.to(dev), adv.to(dev), offsets, ref_logp=refl.to(dev),
                              entropy=ent, mask=keep.to(dev), kl_coef=0.1, entropy_coef=0.01,
                              per_sequence=True)
        d = llmt.token_logprobs_bwd(logits, tgt.reshape(-1), st, p2.dlogp, ent, p2.dentropy)
        x = logits.cpu().double().requires_grad_()
        lg = torch.log_softmax(x, 1)
        h = -(lg.exp() * lg).sum(1)
        (loss_of(oracle_logp(x, tgt.cpu())) - 0.01 * (h * keep).sum() / keep.sum()).backward()
        assert rel_l2(d, x.grad) < 1e-5
    finally:
        ctx.close()
