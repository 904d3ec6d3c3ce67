"""Performance cases of the operators for training all weights on packed sequences: causal
attention over sequences of different lengths, the embedding and its gradient, and an AdamW
step over many tensors with moments in 32 or 8 bits.

Kinds (every one through the public `llmt` binding when `own` is true):

  attn      llmt.packed_attention: causal attention with grouped heads, one call for sequences
            packed one behind another; queries may be the last tokens of longer key sequences
            (a chunk that continues a cache, or single tokens)
  attn_bwd  llmt.packed_attention_bwd: its gradients
  embed     llmt.embedding: rows of a table by token, scaled
  embed_bwd llmt.embedding_bwd: the table's gradient, written whole or added to the one there
  adamw     llmt.adamw_update: one step over a list of tensors, fp32 parameters and their 16-bit
            working copies

The plain forms compute in 32 bits.  8-bit moments are float codes with a power-of-two scale a
block of 256, rounded stochastically by a counter-based generator, so that both sides have the
same random numbers.
"""
import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
V, HIDDEN, KV_DIM, INTER = 151936, 2048, 1024, 6144       # Qwen3-1.7B
# one layer's weights: q, k, v, o, gate, up, down, and its four norms
LAYER = [HIDDEN * HIDDEN, KV_DIM * HIDDEN, KV_DIM * HIDDEN, HIDDEN * HIDDEN, INTER * HIDDEN,
         INTER * HIDDEN, HIDDEN * INTER, HIDDEN, HIDDEN, 128, 128]
BLOCK = 256                                               # 8-bit moments a scale
HP = dict(lr=3e-4, beta1=0.9, beta2=0.999, eps=1e-8, wd=0.01)
MOST_ATTN = 6.0e11                                        # flops of a drawn attention case
MOST_SCORES = 1 << 28


def f32(x):
    """x as the library's float parameters hold it."""
    return float(np.float32(x))


def _llmt():
    root = str(Path(__file__).resolve().parents[1] / "llm.cu_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import llmt
    return llmt


def listed():
    return [
        # eight sequences of a sampling batch, one new token each: latency
        dict(name="attn_step_n8_k9001", kind="attn", dtype="bf16", hd=128, nq=16, nkv=8, n=8,
             tokens=8, mode="step", ctx=9001, key=1),
        # a training micro-batch of answers of different lengths, packed
        dict(name="attn_n16_t8192", kind="attn", dtype="bf16", hd=128, nq=16, nkv=8, n=16,
             tokens=8192, mode="self", ctx=0, key=2),
        # one long document, narrow heads in groups of four
        dict(name="attn_n1_t16384_d64", kind="attn", dtype="f16", hd=64, nq=32, nkv=8, n=1,
             tokens=16384, mode="self", ctx=0, key=3),
        # four pairs of short answers, backward
        dict(name="attn_bwd_n8_t613", kind="attn_bwd", dtype="f16", hd=128, nq=16, nkv=8, n=8,
             tokens=613, mode="self", ctx=0, key=4),
        # the training micro-batch of above, backward
        dict(name="attn_bwd_n16_t8192", kind="attn_bwd", dtype="bf16", hd=128, nq=16, nkv=8, n=16,
             tokens=8192, mode="self", ctx=0, key=2),
        # the headline step's tokens (B1 x S128)
        dict(name="embed_bf16_t128", kind="embed", dtype="bf16", out="bf16", tokens=128, V=V,
             H=HIDDEN, scale=1.0, pad=0.0),
        # a large packed batch on fp32 weights of an odd width, scaled by its root, a tenth padding
        dict(name="embed_f32_t16384_h1037", kind="embed", dtype="f32", out="f32", tokens=16384,
             V=50257, H=1037, scale=32.2, pad=0.1),
        # a short micro-batch added to the accumulated gradient of a tied head
        dict(name="embed_bwd_add_t300", kind="embed_bwd", dtype="bf16", out="f32", tokens=300, V=V,
             H=HIDDEN, scale=1.0, pad=0.0, add=True),
        # a large packed batch, the gradient written whole
        dict(name="embed_bwd_t32768", kind="embed_bwd", dtype="bf16", out="f32", tokens=32768,
             V=50257, H=1024, scale=1.0, pad=0.1, add=False),
        # the norms, biases and other small tensors of a model: many tensors, little work
        dict(name="adamw_32_small200", kind="adamw", bits=32, shapes="small", count=200, grad="f32",
             copy="none", step=7, clip=False),
        # the weights of one layer
        dict(name="adamw_32_layer", kind="adamw", bits=32, shapes="layer", count=1, grad="bf16",
             copy="bf16", step=100, clip=True),
        # two layers with 8-bit moments
        dict(name="adamw_8_layers2", kind="adamw", bits=8, shapes="layer", count=2, grad="bf16",
             copy="bf16", step=100, clip=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn_bwd", "attn_bwd", "embed", "embed_bwd", "adamw"])
    if kind in ("attn", "attn_bwd"):
        while True:
            nq, nkv = rng.choice([(16, 8), (16, 8), (8, 8), (32, 8), (6, 2), (5, 1), (1, 1), (14, 2)])
            mode = rng.choice(["self", "self", "self", "tail", "step"] if kind == "attn" else
                              ["self", "self", "self", "tail"])
            n = _log(rng, 1, 64)
            tokens = n if mode == "step" else _log(rng, 1, 16384)
            ctx = 0 if mode == "self" else _log(rng, max(1, tokens), 65536 if mode == "step" else 16384)
            case = dict(kind=kind, dtype=rng.choice(["bf16", "f16"]), hd=rng.choice([64, 128, 128]),
                        nq=nq, nkv=nkv, n=n, tokens=tokens, mode=mode, ctx=ctx,
                        key=rng.randrange(1 << 20))
            if work(case)["flops"] <= MOST_ATTN:
                return case
    if kind in ("embed", "embed_bwd"):
        H = rng.choice([HIDDEN, _log(rng, 16, 8192)])
        rows = rng.choice([V, _log(rng, 100, 262144)])
        rows = max(100, min(rows, 311_000_000 // H))
        tokens = _log(rng, 1, max(2, min(32768, 33_000_000 // H)))
        low = rng.choice(["bf16", "f16"])
        case = dict(kind=kind, dtype=rng.choice(["f32", low, low]), out="f32", tokens=tokens, V=rows,
                    H=H, scale=rng.choice([1.0, f32(math.sqrt(H))]), pad=rng.choice([0.0, 0.1, 0.4]))
        if rng.random() < 0.5:
            case["out"] = case["dtype"]
        if kind == "embed_bwd":
            case["add"] = rng.random() < 0.5
        return case
    shapes = rng.choice(["small", "layer", "mixed"])
    count = {"small": _log(rng, 1, 400), "layer": rng.choice([1, 1, 2]), "mixed": rng.randint(1, 40)}
    return dict(kind="adamw", bits=rng.choice([8, 32]), shapes=shapes, count=count[shapes],
                grad=rng.choice(["f32", "bf16", "f16"]), copy=rng.choice(["none", "bf16", "f16"]),
                step=_log(rng, 1, 100000), clip=rng.choice([True, False]))


# ---------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _split(total, n, key):
    """n lengths that add up to total, of a few times their spread; some are 0 where n is near it."""
    rng = random.Random(key)
    w = [math.exp(0.7 * rng.gauss(0.0, 1.0)) for _ in range(n)]
    at, s, ends = 0.0, sum(w), [0]
    for x in w:
        at += x
        ends.append(min(total, int(round(total * at / s))))
    ends[-1] = total
    return [b - a for a, b in zip(ends, ends[1:])]


def _lengths(case):
    """Query and key lengths of a case's sequences."""
    n, key = case["n"], case["key"]
    if case["mode"] == "step":
        return [1] * n, [1 + x for x in _split(case["ctx"] - n, n, key)]
    q = _split(case["tokens"], n, key)
    if case["mode"] == "self":
        return q, q
    more = _split(case["ctx"], n, key + 1)
    return q, [a + b for a, b in zip(q, more)]


def _offsets(lengths):
    return np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)


def _pairs(case):
    """(query, key) pairs under the causal mask, whose last query sees every key."""
    ql, kl = _lengths(case)
    return sum(a * (b - a) + a * (a + 1) // 2 for a, b in zip(ql, kl))


def _tensor_sizes(case):
    if case["shapes"] == "layer":
        return LAYER * case["count"]
    rng = random.Random(case["count"])
    if case["shapes"] == "small":
        return [rng.choice([1, 8, 127, 128, 2048, rng.randint(1, 5000)]) for _ in range(case["count"])]
    return [_log(rng, 1, 2_000_000) for _ in range(case["count"])]


def _tokens(case, g):
    """Tokens as text has them: the k-th word with a share of about 1 / k; -1 where padded."""
    u = torch.rand(case["tokens"], generator=g, device="cuda", dtype=torch.float64)
    t = ((case["V"] + 1.0) ** u - 1).to(torch.int32).clamp_(0, case["V"] - 1)
    pad = torch.rand(case["tokens"], generator=g, device="cuda") < case["pad"]
    return torch.where(pad, torch.full_like(t, -1), t)


def prepare(case, seed):
    g = _gen(seed)
    st = dict(case)
    if case["kind"] in ("attn", "attn_bwd"):
        _prepare_attn(case, st, g)
    elif case["kind"] in ("embed", "embed_bwd"):
        st["tok"] = _tokens(case, g)
        if case["kind"] == "embed":
            st["w"] = (0.02 * _randn(g, case["V"], case["H"])).to(DTYPES[case["dtype"]])
        else:
            st["dout"] = (1e-3 * _randn(g, case["tokens"], case["H"])).to(DTYPES[case["dtype"]])
            st["dw"] = torch.zeros(case["V"], case["H"], device="cuda", dtype=DTYPES[case["out"]])
            if case["add"]:
                st["dw"].copy_(1e-4 * _randn(g, case["V"], case["H"]))
    else:
        _prepare_adamw(case, st, g)
    if own:
        st["llmt"] = _llmt()
        if case["kind"] == "adamw":  # the list that a program makes once
            st["list"] = st["llmt"].AdamTensors(st["ps"], st["gs"], st["states"], st["copies"])
    return st


def _prepare_attn(case, st, g):
    ql, kl = _lengths(case)
    nq, nkv, d, dt = case["nq"], case["nkv"], case["hd"], DTYPES[case["dtype"]]
    Tq, Tk = sum(ql), sum(kl)
    st["q_off"] = torch.from_numpy(_offsets(ql)).cuda()
    st["k_off"] = st["q_off"] if case["mode"] == "self" else torch.from_numpy(_offsets(kl)).cuda()
    st["spans"] = list(zip(_offsets(ql).tolist(), ql, _offsets(kl).tolist(), kl))
    if case["mode"] == "self":  # the three parts of one projection's output, as it is
        qkv = _randn(g, Tq, (nq + 2 * nkv) * d).to(dt)
        st["q"] = qkv[:, :nq * d].view(Tq, nq, d)
        st["k"] = qkv[:, nq * d:(nq + nkv) * d].view(Tq, nkv, d)
        st["v"] = qkv[:, (nq + nkv) * d:].view(Tq, nkv, d)
    else:                       # queries of their own, keys and values in caches
        st["q"] = _randn(g, Tq, nq, d).to(dt)
        st["k"] = _randn(g, Tk, nkv, d).to(dt)
        st["v"] = _randn(g, Tk, nkv, d).to(dt)
    if case["kind"] == "attn_bwd":
        st["dout"] = (0.01 * _randn(g, Tq, nq, d)).to(dt)
        st["o"], st["lse"] = _plain_attn(st)


def _prepare_adamw(case, st, g):
    """Parameters, gradients and moments as views of one buffer each, every tensor and every
    tensor's blocks at a place that is a whole number of blocks."""
    sizes = _tensor_sizes(case)
    room = [-(-n // BLOCK) * BLOCK for n in sizes]
    at = np.concatenate([[0], np.cumsum(room)]).tolist()
    N = at[-1]
    st["sizes"], st["at"] = sizes, at
    gdt = DTYPES[case["grad"]]

    def views(flat):
        return [flat[a:a + n] for a, n in zip(at, sizes)]
    st["p"] = 0.02 * _randn(g, N)
    st["ps"] = views(st["p"])
    # gradients whose size differs from tensor to tensor and from element to element
    gr = 1e-3 * _randn(g, N) * torch.exp(0.5 * _randn(g, N))
    st["gs"] = views(gr.to(gdt))
    m = 3e-4 * _randn(g, N) * torch.exp(0.5 * _randn(g, N))
    v = 1e-6 * torch.exp(_randn(g, N))
    st["copy"] = None if case["copy"] == "none" else torch.zeros(N, device="cuda",
                                                                 dtype=DTYPES[case["copy"]])
    st["copies"] = None if st["copy"] is None else views(st["copy"])
    st["factor"] = torch.full((1,), 0.7, device="cuda") if case["clip"] else None
    # the space behind a tensor's end holds nothing
    for flat in (m, v):
        for a, n, r in zip(at, sizes, room):
            flat[a + n:a + r] = 0
    if case["bits"] == 32:
        st["m"], st["v"] = m, v
        st["states"] = [(a, b, None, None) for a, b in zip(views(m), views(v))]
        return
    half = torch.full((N // BLOCK, BLOCK), 1 << 15, device="cuda", dtype=torch.int64)
    mc, me = _encode(m.view(-1, BLOCK), 15, half)
    vc, ve = _encode(v.view(-1, BLOCK), 31, half)
    st["m"], st["v"] = mc.view(-1), vc.view(-1)
    st["me"], st["ve"] = me, ve                  # a byte a block
    st["states"] = [(a, b, me[s // BLOCK:(s + r) // BLOCK], ve[s // BLOCK:(s + r) // BLOCK])
                    for a, b, s, r in zip(views(st["m"]), views(st["v"]), at, room)]


# ---------------------------------------------------------------- plain forms

def _scores(q, k, scale, first, shift):
    """Masked fp32 scores [nkv, group * rows, keys] of query rows from `first` on."""
    rows, nq, d = q.shape
    nkv = k.shape[1]
    qs = q.float().view(rows, nkv, nq // nkv, d).permute(1, 2, 0, 3).reshape(nkv, -1, d)
    s = torch.matmul(qs, k.float().permute(1, 2, 0).contiguous()) * scale
    at = torch.arange(rows, device=q.device) + (first + shift)
    hide = torch.arange(k.shape[0], device=q.device)[None, :] > at[:, None]
    return qs, s.masked_fill_(hide.repeat(nq // nkv, 1)[None], -math.inf)


def _rows_back(x, rows, nq):
    """[nkv, group * rows, d] -> [rows, nq, d]."""
    nkv, _, d = x.shape
    return x.view(nkv, nq // nkv, rows, d).permute(2, 0, 1, 3).reshape(rows, nq, d)


def _chunks(ql, kl, nq):
    """Query ranges whose scores fit a bound."""
    step = max(1, min(ql, MOST_SCORES // max(1, kl * nq)))
    return [(a, min(ql, a + step)) for a in range(0, ql, step)]


def _plain_attn(st):
    q, k, v = st["q"], st["k"], st["v"]
    nq, d = q.shape[1:]
    scale = 1.0 / math.sqrt(d)
    o = torch.zeros(q.shape, device="cuda", dtype=q.dtype)
    lse = torch.full((q.shape[0], nq), -math.inf, device="cuda")
    for q0, ql, k0, kl in st["spans"]:
        ks, vs = k[k0:k0 + kl], v[k0:k0 + kl].float().transpose(0, 1)
        for a, b in _chunks(ql, kl, nq):
            _, s = _scores(q[q0 + a:q0 + b], ks, scale, a, kl - ql)
            m = s.amax(-1, keepdim=True)
            p = (s - m).exp_()
            l = p.sum(-1, keepdim=True)
            o[q0 + a:q0 + b] = _rows_back(torch.matmul(p, vs) / l, b - a, nq).to(q.dtype)
            lse[q0 + a:q0 + b] = _rows_back(m + l.log(), b - a, nq)[..., 0]
    return o, lse


def _plain_attn_bwd(st):
    q, k, v, o, lse, do = (st[x] for x in ("q", "k", "v", "o", "lse", "dout"))
    nq, d = q.shape[1:]
    nkv, scale = k.shape[1], 1.0 / math.sqrt(q.shape[2])
    dq = torch.zeros(q.shape, device="cuda", dtype=q.dtype)
    dk, dv = (torch.zeros(k.shape, device="cuda", dtype=q.dtype) for _ in range(2))

    def heads(x, a, b):
        return x[a:b].float().view(b - a, nkv, nq // nkv, -1).permute(1, 2, 0, 3).reshape(
            nkv, (b - a) * (nq // nkv), -1)
    for q0, ql, k0, kl in st["spans"]:
        ks, vs = k[k0:k0 + kl], v[k0:k0 + kl].float()
        gk = torch.zeros(nkv, kl, d, device="cuda")
        gv = torch.zeros(nkv, kl, d, device="cuda")
        for a, b in _chunks(ql, kl, nq):
            qs, s = _scores(q[q0 + a:q0 + b], ks, scale, a, kl - ql)
            p = (s - heads(lse, q0 + a, q0 + b)).exp_()
            dos = heads(do, q0 + a, q0 + b)
            delta = (dos * heads(o, q0 + a, q0 + b)).sum(-1, keepdim=True)
            gv += torch.matmul(p.transpose(1, 2), dos)
            ds = (torch.matmul(dos, vs.permute(1, 2, 0).contiguous()) - delta) * p
            gk += torch.matmul(ds.transpose(1, 2), qs) * scale
            g = torch.matmul(ds, ks.float().transpose(0, 1)) * scale
            dq[q0 + a:q0 + b] = _rows_back(g, b - a, nq).to(q.dtype)
        dk[k0:k0 + kl] = gk.transpose(0, 1).to(q.dtype)
        dv[k0:k0 + kl] = gv.transpose(0, 1).to(q.dtype)
    return dq, dk, dv


def _plain_embed(st):
    t = st["tok"].long()
    keep = ((t >= 0) & (t < st["V"]))[:, None]
    x = st["w"][t.clamp(0, st["V"] - 1)].float() * f32(st["scale"])
    return torch.where(keep, x, torch.zeros_like(x)).to(DTYPES[st["out"]])


def _plain_embed_bwd(st):
    t = st["tok"].long()
    keep = (t >= 0) & (t < st["V"])
    d = st["dout"].float() * keep[:, None]
    g = torch.zeros(st["V"], st["H"], device="cuda")
    g.index_add_(0, t.clamp(0, st["V"] - 1), d)
    g *= f32(st["scale"])
    if st["add"]:
        g += st["dw"]
    st["dw"].copy_(g)
    return st["dw"]


def _encode(x, top, rnd):
    """Blocks x [nb, 256] as 8-bit float codes: (codes, exponents), uint8.  A block's scale is the
    power of two that brings its largest value below 1.875; below it a code has `top` binades of
    eight steps, then zero.  rnd, 16 bits: the share of a step that rounds up."""
    bits = x.abs().amax(1).view(torch.int32)
    e = (bits >> 23) + ((bits & 0x7FFFFF) > 0x700000).int()
    e = torch.where(e >= 254, 255, e.clamp(min=1))
    down = ((254 - e.clamp(max=253)) << 23).view(torch.float32)[:, None]
    y = (x.abs() * down) * 2.0 ** (top - 127)
    code = ((y.view(torch.int32) + (rnd << 4).int()) >> 20)
    if top == 15:
        code = code | ((x < 0).int() << 7)
    else:
        code = torch.maximum(code, (x > 0).int())
    return torch.where((e == 255)[:, None], 0, code).to(torch.uint8), e.to(torch.uint8)


def _decode(code, e, top):
    c, e = code.int(), e.int()
    mag = ((c & (127 if top == 15 else 255)) << 20).view(torch.float32) * 2.0 ** (127 - top)
    mag = mag * (e.clamp(max=254) << 23).view(torch.float32)[:, None]
    if top == 15:
        mag = torch.where(c >= 128, -mag, mag)
    return torch.where((e == 255)[:, None], math.nan, mag)


M64 = (1 << 64) - 1


def _mix(x):
    """The generator's 64-bit mix of a Python integer."""
    x = (x + 0x9E3779B97F4A7C15) & M64
    x = ((x ^ (x >> 30)) * 0xBF58476D1CE4E5B9) & M64
    x = ((x ^ (x >> 27)) * 0x94D049BB133111EB) & M64
    return x ^ (x >> 31)


def _signed(x):
    return x - (1 << 64) if x >> 63 else x


def _mix_t(x):
    """The same on int64 tensors."""
    def shr(v, n):
        return (v >> n) & ((1 << (64 - n)) - 1)
    x = x + _signed(0x9E3779B97F4A7C15)
    x = (x ^ shr(x, 30)) * _signed(0xBF58476D1CE4E5B9)
    x = (x ^ shr(x, 27)) * _signed(0x94D049BB133111EB)
    return x ^ shr(x, 31)


def _draws(blocks, seed, step, tensor):
    """16-bit draws for m and v of a tensor's elements, [blocks, 256] each: one 64-bit value of
    the generator for two elements."""
    key = _signed(_mix(_mix(seed) ^ ((step << 32) + tensor)))
    x = _mix_t(torch.arange(blocks * BLOCK // 2, device="cuda") + key)
    m = torch.stack([x & 0xFFFF, (x >> 32) & 0xFFFF], 1)
    v = torch.stack([(x >> 16) & 0xFFFF, (x >> 48) & 0xFFFF], 1)
    return m.view(blocks, BLOCK), v.view(blocks, BLOCK)


def _padded(x, blocks):
    out = torch.zeros(blocks * BLOCK, device="cuda")
    out[:x.numel()] = x
    return out.view(blocks, BLOCK)


def _adamw_outputs(st, values):
    return [st["p"], st["copy"], *values]


def _plain_adamw(st):
    b1, b2, lr, eps, wd = (f32(HP[x]) for x in ("beta1", "beta2", "lr", "eps", "wd"))
    c1, c2 = f32(1 - b1), f32(1 - b2)
    bc1, bc2 = 1 - b1 ** st["step"], 1 - b2 ** st["step"]
    vals = [torch.zeros_like(st["p"]) for _ in range(2)] if st["bits"] == 8 else [st["m"], st["v"]]
    for i, n in enumerate(st["sizes"]):
        p, g = st["ps"][i], st["gs"][i].float()
        mc, vc, me, ve = st["states"][i]
        if st["factor"] is not None:
            g = g * st["factor"]
        if me is not None:
            a, nb = st["at"][i], me.shape[0]
            codes = [st[x][a:a + nb * BLOCK].view(nb, BLOCK) for x in ("m", "v")]
            m = _decode(codes[0], me, 15).view(-1)[:n]
            v = _decode(codes[1], ve, 31).view(-1)[:n]
        else:
            m, v = mc, vc
        m2 = m * b1 + g * c1
        v2 = v * b2 + (g * c2) * g
        p.copy_(p * f32(1 - lr * wd) - (lr / bc1) * m2 / ((v2 / bc2).sqrt() + eps))
        if st["copies"] is not None:
            st["copies"][i].copy_(p)
        if me is None:
            mc.copy_(m2)
            vc.copy_(v2)
            continue
        rm, rv = _draws(nb, 1, st["step"], i)
        for x, e, y, top, r, out in ((codes[0], me, m2, 15, rm, vals[0]),
                                     (codes[1], ve, v2, 31, rv, vals[1])):
            code, ex = _encode(_padded(y, nb), top, r)
            code.view(-1)[n:] = 0
            x.copy_(code)
            e.copy_(ex)
            out[a:a + n] = _decode(code, ex, top).view(-1)[:n]
    return _adamw_outputs(st, vals)


# ---------------------------------------------------------------- one pass

def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_plain(st):
    return {"attn": _plain_attn, "attn_bwd": _plain_attn_bwd, "embed": _plain_embed,
            "embed_bwd": _plain_embed_bwd, "adamw": _plain_adamw}[st["kind"]](st)


def _run_own(st):
    llmt, kind = st["llmt"], st["kind"]
    if kind == "attn":
        return llmt.packed_attention(st["q"], st["k"], st["v"], st["q_off"], st["k_off"])
    if kind == "attn_bwd":
        return llmt.packed_attention_bwd(st["q"], st["k"], st["v"], st["o"], st["lse"], st["dout"],
                                         st["q_off"], st["k_off"])
    if kind == "embed":
        return llmt.embedding(st["tok"], st["w"], scale=st["scale"], out_dtype=DTYPES[st["out"]])
    if kind == "embed_bwd":
        return llmt.embedding_bwd(st["tok"], st["dout"], st["dw"], scale=st["scale"],
                                  accumulate=st["add"])
    llmt.adamw_update(st["list"], llmt.hparams(**HP), st["step"], grad_scale=st["factor"], seed=1)
    if st["bits"] == 32:
        return _adamw_outputs(st, [st["m"], st["v"]])
    return _adamw_outputs(st, llmt.adamw_moments((st["m"], st["v"], st["me"], st["ve"])))


# ---------------------------------------------------------------- work

def _size(name):
    return 4 if name == "f32" else 2


def work(case):
    if case["kind"] in ("attn", "attn_bwd"):
        ql, kl = _lengths(case)
        Tq, Tk = sum(ql), sum(kl)
        q = Tq * case["nq"] * case["hd"] * 2
        kv = 2 * Tk * case["nkv"] * case["hd"] * 2
        lse = 4 * Tq * case["nq"]
        flops = 4 * case["hd"] * case["nq"] * _pairs(case)
        if case["kind"] == "attn":
            return {"bytes": 2 * q + kv + lse, "flops": flops}
        return {"bytes": 4 * q + 2 * kv + lse, "flops": 2.5 * flops}
    if case["kind"] in ("embed", "embed_bwd"):
        T, H = case["tokens"], case["H"]
        # the distinct words among T of a share of 1 / k each
        ln = math.log(case["V"] + 1.0)
        kept = T * (1 - case["pad"])
        k = np.arange(1, case["V"] + 1, dtype=np.float64)
        seen = float((-np.expm1(kept * np.log1p(-np.log1p(1 / k) / ln))).sum())
        if case["kind"] == "embed":
            return {"bytes": 4 * T + seen * H * _size(case["dtype"]) + T * H * _size(case["out"]),
                    "flops": kept * H}
        out = _size(case["out"])
        rows = 2 * seen if case["add"] else case["V"]
        return {"bytes": 4 * T + kept * H * _size(case["dtype"]) + rows * H * out,
                "flops": kept * H}
    n = sum(_tensor_sizes(case))
    moments = 16 if case["bits"] == 32 else 4 + 4 / BLOCK
    copy = 0 if case["copy"] == "none" else 2
    values = 0 if case["bits"] == 32 else 8   # 8-bit moments are returned as what they stand for
    return {"bytes": n * (8 + _size(case["grad"]) + moments + copy + values), "flops": 16 * n}


# ---------------------------------------------------------------- in 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "attn":
        return _exact_attn(st)
    if case["kind"] == "attn_bwd":
        return _exact_attn_bwd(st)
    if case["kind"] == "embed":
        out = torch.zeros(case["tokens"], case["H"], device="cuda", dtype=torch.float64)
        ok = (st["tok"] >= 0).nonzero()[:, 0]
        out[ok] = st["w"].index_select(0, st["tok"][ok]).double() * f32(case["scale"])
        return out
    if case["kind"] == "embed_bwd":
        ok = (st["tok"] >= 0).nonzero()[:, 0]
        out = st["dw"].double() if case["add"] else torch.zeros(
            case["V"], case["H"], device="cuda", dtype=torch.float64)
        out.index_add_(0, st["tok"][ok].long(), st["dout"][ok].double() * f32(case["scale"]))
        return out
    return _exact_adamw(st)


def _exact_heads(st):
    """(sequence's rows of q, of k, query head, its KV head, allowed pairs) one after another."""
    nq, nkv = st["q"].shape[1], st["k"].shape[1]
    for q0, ql, k0, kl in st["spans"]:
        if ql:
            see = torch.ones(ql, kl, dtype=torch.bool, device="cuda").tril_(kl - ql)
            for h in range(nq):
                yield slice(q0, q0 + ql), slice(k0, k0 + kl), h, h * nkv // nq, see


def _exact_attn(st):
    q, k, v = st["q"], st["k"], st["v"]
    o = torch.zeros(q.shape, device="cuda", dtype=torch.float64)
    lse = torch.full(q.shape[:2], -math.inf, device="cuda", dtype=torch.float64)
    for rows, keys, h, j, see in _exact_heads(st):
        s = q[rows, h].double() @ k[keys, j].double().t() / math.sqrt(q.shape[2])
        s[~see] = -math.inf
        lse[rows, h] = torch.logsumexp(s, 1)
        o[rows, h] = torch.softmax(s, 1) @ v[keys, j].double()
    return o, lse


def _exact_attn_bwd(st):
    q, k, v = st["q"], st["k"], st["v"]
    root = math.sqrt(q.shape[2])
    dq = torch.zeros(q.shape, device="cuda", dtype=torch.float64)
    dk, dv = (torch.zeros(k.shape, device="cuda", dtype=torch.float64) for _ in range(2))
    for rows, keys, h, j, see in _exact_heads(st):
        qh, kh, do = q[rows, h].double(), k[keys, j].double(), st["dout"][rows, h].double()
        p = torch.exp(qh @ kh.t() / root - st["lse"][rows, h].double()[:, None]) * see
        dv[keys, j] += p.t() @ do
        dp = do @ v[keys, j].double().t()
        ds = p * (dp - (do * st["o"][rows, h].double()).sum(1)[:, None]) / root
        dq[rows, h] = ds @ kh
        dk[keys, j] += ds.t() @ qh
    return dq, dk, dv


def _exact_adamw(st):
    b1, b2, lr, eps, wd = (f32(HP[x]) for x in ("beta1", "beta2", "lr", "eps", "wd"))
    t = st["step"]
    P, M, W = st["p"].double(), st["p"].double() * 0, st["p"].double() * 0
    if st["bits"] == 8:
        m0 = _decode(st["m"].view(-1, BLOCK), st["me"], 15).view(-1).double()
        v0 = _decode(st["v"].view(-1, BLOCK), st["ve"], 31).view(-1).double()
    else:
        m0, v0 = st["m"].double(), st["v"].double()
    for a, n, g in zip(st["at"], st["sizes"], st["gs"]):
        s = slice(a, a + n)
        g = g.double() * (1.0 if st["factor"] is None else st["factor"].double())
        M[s] = b1 * m0[s] + (1 - b1) * g
        W[s] = b2 * v0[s] + (1 - b2) * g * g
        step = (M[s] / (1 - b1 ** t)) / ((W[s] / (1 - b2 ** t)).sqrt() + eps)
        P[s] -= lr * wd * P[s] + lr * step
    copy = None
    if st["copy"] is not None:
        copy = torch.zeros_like(P)
        for a, n in zip(st["at"], st["sizes"]):
            copy[a:a + n] = P[a:a + n]
    # 8-bit moments are defined by their rounding: they have no value of 64 bits
    return [P, copy, None, None] if st["bits"] == 8 else [P, copy, M, W]
