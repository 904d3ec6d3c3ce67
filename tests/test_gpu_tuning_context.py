"""GPU: log-probabilities and Muon on a context, where calls meet that do not belong
together: refused weights, other streams, another optimiser's state."""
import copy
import ctypes as C

import pytest
import torch

import llmt
from helpers import SMALL, small_problem, upload_model
from oracle.configs import quantize_model_int8

pytestmark = pytest.mark.gpu


def context(dev, W, ad, batch, seq_len, stream=None):
    ctx = llmt.Context(llmt.make_dims(SMALL), max_batch=batch, seq_len=seq_len, stream=stream)
    upload_model(ctx, W, dev)
    ctx.lora_set("param", llmt.flatten_adapters(ad).to(dev))
    return ctx


@pytest.mark.parametrize("weights", ["f16", "i8"])
def test_layer_setters_and_the_backward(dev, weights):
    """A setter that refuses its arguments changes nothing; one that takes them ends the
    stashes of the last forward."""
    W, ad, tok, tgt = small_problem()
    B, S = tok.shape
    tok, tgt = tok.to(dev), tgt.to(dev)
    L = llmt.lib()
    f = lambda t: t.float().to(dev).contiguous()
    norms = [f(t) for t in (W.layers[0].attn_norm, W.layers[0].ffn_norm, W.layers[0].q_norm,
                            W.layers[0].k_norm)]
    names = ("wq", "wk", "wv", "wo", "w_gate", "w_up", "w_down")
    if weights == "i8":
        W, qs = quantize_model_int8(copy.deepcopy(W))
        ctx = llmt.Context(llmt.make_dims(SMALL), B, S, int8=True)
        q = [[torch.from_numpy(qs[(l, n)][0]).to(dev) for n in names] for l in range(2)]
        s = [[torch.from_numpy(qs[(l, n)][1]).to(dev) for n in names] for l in range(2)]

        def put(l, norms, of=None):
            of = l if of is None else of
            arr = lambda ts: (llmt.vp * 7)(*(t.data_ptr() for t in ts))
            return L.llmt_set_layer_i8(ctx.h, l, arr(q[of]), arr(s[of]), *map(llmt.ptr, norms))
    else:
        ctx = llmt.Context(llmt.make_dims(SMALL), B, S)
        h = [[getattr(lw, n).half().to(dev).contiguous() for n in names] for lw in W.layers]

        def put(l, norms, of=None):
            return L.llmt_set_layer_f16(ctx.h, l, *map(llmt.ptr, h[l if of is None else of]),
                                        *map(llmt.ptr, norms))
    try:
        assert put(0, norms) == 0 and put(1, norms) == 0
        ctx.set_embed_f16(W.embed.half().to(dev), f(W.final_norm))
        ctx.lora_set("param", llmt.flatten_adapters(ad).to(dev))
        d = torch.linspace(-1, 1, B * S, device=dev)
        want = ctx.forward_logprobs(tok, tgt)
        ctx.backward_logprobs(d)
        grad = ctx.lora_get("grad")
        for k in range(4):
            bad = list(norms)
            bad[k] = None
            assert put(0, bad, of=1) == llmt.LLMT_ERR_ARG      # the other layer's matrices
            ctx.backward_logprobs(d)
            assert torch.equal(ctx.lora_get("grad"), grad)
            assert torch.equal(ctx.forward_logprobs(tok, tgt), want)
        assert put(1, norms) == 0
        assert L.llmt_backward_logprobs(ctx.h, llmt.ptr(d)) == llmt.LLMT_ERR_STATE
        assert torch.equal(ctx.forward_logprobs(tok, tgt), want)
    finally:
        ctx.close()


def busy(seconds=0.03):
    """Work of about that long on the current stream."""
    a = torch.zeros(4096, 4096, device="cuda")
    for _ in range(int(seconds / 1e-3)):
        torch.mm(a, a, out=torch.empty_like(a))


@pytest.mark.parametrize("where", ["side", "given", "same"])
def test_calls_follow_the_current_stream(dev, where):
    """A preference step where torch's current stream, the context's or both are a stream
    that nothing else is ordered with, and inputs are written late: as on the default one."""
    W, ad, tok, tgt = small_problem()
    B, S = tok.shape
    flat = llmt.flatten_adapters(ad).to(dev)
    tok, tgt = tok.to(dev), tgt.to(dev)
    offsets = torch.arange(0, B * S + 1, S, dtype=torch.int32, device=dev)
    ref_lp = torch.full((B * S,), -7.0, device=dev)

    def step(ctx, late):
        def now(t):                               # t, written as late as its stream gets to it
            if not late:
                return t
            x = torch.zeros_like(t)
            torch.cuda.current_stream().synchronize()
            busy()
            return x.copy_(t)

        ctx.lora_set("param", now(flat))
        lp = ctx.forward_logprobs(now(tok), now(tgt))
        if late:
            busy()
        d = llmt.preference_loss(lp, ref_lp, offsets, beta=0.5)[3]
        ctx.backward_logprobs(now(d))
        grad = ctx.lora_get("grad")
        logits = ctx.logits(B * S)
        loss = ctx.forward_backward(now(tok), now(tgt))
        return lp, d, grad, logits, torch.tensor(loss)

    ctx = context(dev, W, ad, B, S)
    try:
        want = step(ctx, False)
        torch.cuda.synchronize()
    finally:
        ctx.close()
    side = torch.cuda.Stream()
    ctx = context(dev, W, ad, B, S, stream=None if where == "side" else side)
    try:
        torch.cuda.synchronize()
        with torch.cuda.stream(torch.cuda.default_stream() if where == "given" else side):
            got = step(ctx, True)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    finally:
        ctx.close()


def test_muon_state_is_not_adamws(dev, tmp_path):
    """Momentum of Muon's in the M arena, stepped there or loaded, is no AdamW state: AdamW
    refuses until the arena is set anew.  Saved and loaded, Muon continues bit for bit."""
    W, ad, tok, tgt = small_problem()
    B, S = tok.shape
    tok, tgt = tok.to(dev), tgt.to(dev)
    L, hp, adam = llmt.lib(), llmt.muon_hparams(lr=1e-3), llmt.hparams()
    flat = llmt.flatten_adapters(ad).to(dev)
    ctx = context(dev, W, ad, B, S)

    def adamw_refused():
        before = ctx.lora_get("param"), ctx.lora_get("m")
        for graph in (False, True):
            ctx.set_graph(graph)
            with pytest.raises(llmt.LlmtError, match="Muon"):
                ctx.step(tok, tgt, adam, 3)
        ctx.set_graph(False)
        assert L.llmt_adamw(ctx.h, C.byref(adam), 3) == llmt.LLMT_ERR_STATE
        with pytest.raises(llmt.LlmtError, match="Muon"):
            ctx.profile_kernels(tok, tgt, adam, 3, reps=1)
        assert torch.equal(ctx.lora_get("param"), before[0])
        assert torch.equal(ctx.lora_get("m"), before[1])

    try:
        ctx.step(tok, tgt, adam, 1)
        ctx.lora_save_state(tmp_path, 1)
        assert (tmp_path / "lora_step1_adamw.bin").read_bytes()[:8] == b"LLMTADAM"
        m1, p1 = ctx.lora_get("m"), ctx.lora_get("param")
        ctx.step(tok, tgt, adam, 2)
        p2 = ctx.lora_get("param")
        ctx.lora_set("m", torch.zeros_like(m1))
        ctx.forward_backward(tok, tgt)
        ctx.muon(hp)
        adamw_refused()
        ctx.lora_save_state(tmp_path, 2)
        m2, pm = ctx.lora_get("m"), ctx.lora_get("param")
        ctx.forward_backward(tok, tgt)
        ctx.muon(hp)
        want = ctx.lora_get("param")
        # AdamW's state again: its next step as it was
        ctx.lora_set("param", p1)
        ctx.lora_load_state(tmp_path, 1)
        assert torch.equal(ctx.lora_get("m"), m1)
        ctx.step(tok, tgt, adam, 2)
        assert torch.equal(ctx.lora_get("param"), p2)
        # Muon's in a context of its own
        ctx.close()
        ctx = context(dev, W, ad, B, S)
        ctx.lora_set("param", pm)
        ctx.lora_load_state(tmp_path, 2)
        assert torch.equal(ctx.lora_get("m"), m2)
        adamw_refused()
        ctx.forward_backward(tok, tgt)
        ctx.muon(hp)
        assert torch.equal(ctx.lora_get("param"), want)
        # the arena set anew
        ctx.lora_set("param", flat)
        adamw_refused()
        ctx.lora_set("m", torch.zeros_like(m1))
        ctx.step(tok, tgt, adam, 1)
        ctx.muon(hp)
        ctx.lora_init(1, 0.02, 0.0)
        ctx.step(tok, tgt, adam, 1)
    finally:
        ctx.close()
