"""Performance cases of the tuning operators: token log-probabilities over a vocabulary,
the preference and policy losses on them, and the orthogonalised (Muon) update of adapters.

Kinds (every one through the public `llmt` binding when `own` is true):

  logp      llmt.token_logprobs: log-probability of each row's target, the softmax
            statistics and, where wanted, the entropy
  logp_bwd  llmt.token_logprobs_bwd: the gradient of the logits from the gradients of the
            log-probabilities (and entropies)
  pref      llmt.preference_loss: paired log-ratio loss of (chosen, rejected) sequences, the
            rewards and the gradient of every token's log-probability
  policy    llmt.policy_loss: clipped policy loss with a KL term and an entropy bonus, its
            statistics and its gradients
  ortho     llmt.orthogonalize: Newton-Schulz orthogonalisation of a stack of matrices
  muon      llmt.muon_update: momentum, orthogonalisation and the update of a whole arena

The plain forms compute in 32 bits, and in 64 where 32 lose what matters: the sums over a
sequence, and the ratios that are compared with the clip borders.
"""
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

V = 151936                                    # Qwen3's vocabulary
RANK, HIDDEN, KV_DIM, LAYERS = 16, 2048, 1024, 28
# the adapters of one layer, q, k, v, o: A [rank, in], B [out, rank]
LAYER_SHAPES = [(RANK, HIDDEN), (HIDDEN, RANK), (RANK, HIDDEN), (KV_DIM, RANK),
                (RANK, HIDDEN), (KV_DIM, RANK), (RANK, HIDDEN), (HIDDEN, RANK)]
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
NS = (3.4445, -4.7750, 2.0315)                # the quintic's coefficients
EPS = 1e-7


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
        # one sampled token scored by its model: a single row, latency
        dict(name="logp_f32_r1_v151936", kind="logp", dtype="f32", rows=1, V=V, skip=0.0,
             entropy=False, temperature=1.0),
        # the large-batch configuration (B8 x S512) scored, a quarter of it prompt or padding
        dict(name="logp_f32_r4096_v151936", kind="logp", dtype="f32", rows=4096, V=V, skip=0.25,
             entropy=False, temperature=1.0),
        # the gradient at the headline step's size (B1 x S128); the last row has no target
        dict(name="logp_bwd_f32_r128_v151936", kind="logp_bwd", dtype="f32", rows=128, V=V,
             skip=0.008, entropy=False, temperature=1.0),
        # half-precision logits over a vocabulary of odd length, sampled at a temperature, with
        # the entropy bonus
        dict(name="logp_bwd_bf16_r1000_v50257", kind="logp_bwd", dtype="bf16", rows=1000, V=50257,
             skip=0.3, entropy=True, temperature=0.7),
        # a micro-batch of four pairs of answers
        dict(name="pref_n4_s300", kind="pref", n=4, S=300, loss="sigmoid", beta=0.1, smooth=0.0,
             margin=0.0, average=False, ref=True, mask=True),
        # a data set's epoch of precomputed pairs, length-normalised with a margin
        dict(name="pref_n2048_s700", kind="pref", n=2048, S=700, loss="sigmoid", beta=2.0,
             smooth=0.1, margin=0.5, average=True, ref=False, mask=True),
        # eight sampled answers to one prompt, an advantage for each
        dict(name="policy_n8_s200", kind="policy", n=8, S=200, per_sequence=True, mean="token",
             low=0.2, high=0.2, kl=0.04, ent=0.0, mask=True),
        # a rollout batch with an advantage for each token, mean over the sequences
        dict(name="policy_n512_s1800", kind="policy", n=512, S=1800, per_sequence=False,
             mean="sequence", low=0.2, high=0.28, kl=0.02, ent=0.01, mask=True),
        # one adapter's update, latency
        dict(name="ortho_1x16x2048", kind="ortho", count=1, rows=16, cols=2048, steps=5),
        # adapters of a higher rank on a wide projection, tall
        dict(name="ortho_28x12288x64", kind="ortho", count=28, rows=12288, cols=64, steps=5),
        # one layer's adapters
        dict(name="muon_1layer_r16", kind="muon", layers=1, shapes="qwen", rank=16, nesterov=True,
             scale="rms"),
        # the whole adapter arena of the headline model
        dict(name="muon_28layers_r16", kind="muon", layers=LAYERS, shapes="qwen", rank=16,
             nesterov=True, scale="rms"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["logp", "logp_bwd", "pref", "policy", "ortho", "muon"])
    if kind in ("logp", "logp_bwd"):
        v = rng.choice([V, V, _log(rng, 32, 262144)])
        most = 200_000_000 // v
        return dict(kind=kind, dtype=rng.choice(["f32", "f16", "bf16"]),
                    rows=_log(rng, 1, max(2, min(8192, most))), V=v,
                    skip=rng.choice([0.0, 0.1, 0.5]), entropy=rng.choice([True, False]),
                    temperature=rng.choice([1.0, 0.8, 1.3]))
    if kind == "pref":
        S = _log(rng, 1, 4096)
        return dict(kind=kind, n=_log(rng, 1, max(2, min(2048, 1_400_000 // S))), S=S,
                    loss=rng.choice(["sigmoid", "hinge", "square"]),
                    beta=rng.choice([0.05, 0.1, 0.5]), smooth=rng.choice([0.0, 0.1]),
                    margin=rng.choice([0.0, 0.3]), average=rng.choice([True, False]),
                    ref=rng.choice([True, False]), mask=rng.choice([True, False]))
    if kind == "policy":
        S = _log(rng, 1, 4096)
        return dict(kind=kind, n=_log(rng, 1, max(2, min(2048, 900_000 // S))), S=S,
                    per_sequence=rng.choice([True, False]), mean=rng.choice(["token", "sequence"]),
                    low=rng.choice([0.1, 0.2]), high=rng.choice([0.2, 0.28]),
                    kl=rng.choice([0.0, 0.04]), ent=rng.choice([0.0, 0.01]),
                    mask=rng.choice([True, False]))
    if kind == "ortho":
        r = rng.choice([1, 4, 8, 16, 16, 16, 24, 32, 33, 64])
        n = max(r, _log(rng, 16, 16384))
        count = _log(rng, 1, max(2, min(224, 6_000_000 // (r * n))))
        return dict(kind=kind, count=count, rows=r, cols=n, steps=rng.choice([4, 5, 6])) \
            if rng.random() < 0.5 else \
            dict(kind=kind, count=count, rows=n, cols=r, steps=rng.choice([4, 5, 6]))
    return dict(kind=kind, layers=rng.randint(1, LAYERS), shapes=rng.choice(["qwen", "other"]),
                rank=rng.choice([8, 16, 16, 32]), nesterov=rng.choice([True, False]),
                scale=rng.choice(["rms", "shape"]))


# ---------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _rand(g, *shape):
    return torch.rand(shape, generator=g, device="cuda")


def _shapes(case):
    """The matrices of one layer of a muon case."""
    r = case["rank"]
    if case["shapes"] == "qwen":
        return [tuple(r if d == RANK else d for d in s) for s in LAYER_SHAPES]
    return [(r, 896), (896, r), (r, 896), (128, r)]


def _sequences(case, g, count):
    """`count` ragged sequences of up to S tokens behind one another, in an order of the seed's:
    offsets [count + 1] and the number of tokens.  In a longer list every eighth is empty."""
    n = [0 if count >= 16 and i % 8 == 5 else math.ceil(case["S"] * (0.3 + 0.7 * (i + 1) / count))
         for i in range(count)]
    n = torch.tensor(n, device="cuda")[torch.randperm(count, generator=g, device="cuda")]
    off = torch.zeros(count + 1, dtype=torch.int32, device="cuda")
    off[1:] = n.cumsum(0)
    return off, int(off[-1])


def _logits(case, seed):
    g = _gen(seed)
    rows, v, dt = case["rows"], case["V"], DTYPES[case["dtype"]]
    logits = torch.empty(rows, v, dtype=dt, device="cuda")
    step = max(1, (1 << 28) // v)
    for i in range(0, rows, step):
        # a trained model's logits: a spread of a few units and a few likely tokens
        x = _randn(g, min(step, rows - i), v).mul_(2.5)
        logits[i:i + step] = x.to(dt)
    tgt = torch.randint(0, v, (rows,), generator=g, device="cuda", dtype=torch.int32)
    logits[torch.arange(rows, device="cuda"), tgt.long()] += (4.0 + 3.0 * _randn(g, rows)).to(dt)
    nskip = math.ceil(case["skip"] * rows) if rows > 1 else 0
    tgt[torch.randperm(rows, generator=g, device="cuda")[:nskip]] = -1
    return g, logits, tgt


def prepare(case, seed):
    kind = case["kind"]
    st = dict(case=case)
    if kind in ("logp", "logp_bwd"):
        g, st["logits"], st["targets"] = _logits(case, seed)
        if kind == "logp_bwd":  # what the forward left, and the loss's gradients
            rows = case["rows"]
            stats, ent = [], []
            for i in range(0, rows, 256):
                x = st["logits"][i:i + 256].double() * f32(1.0 / case["temperature"])
                mx = x.amax(1)
                e = (x - mx[:, None]).exp_()
                s = e.sum(1)
                stats.append(torch.stack([mx.float(), (s.log() + (mx - mx.float().double())).float()], 1))
                ent.append((s.log() - (e * (x - mx[:, None])).sum(1) / s).float())
                del x, e
            st["stats"] = torch.cat(stats)
            st["dlogp"] = _randn(g, rows) / rows
            if case["entropy"]:
                st["entropy"] = torch.cat(ent)
                st["dentropy"] = torch.full((rows,), -0.01 / rows, device="cuda")
    elif kind == "pref":
        g = _gen(seed)
        st["offsets"], T = _sequences(case, g, 2 * case["n"])
        st["logp"] = -_randn(g, T).abs() * 1.5
        if case["ref"]:
            st["ref"] = st["logp"] + 0.2 * _randn(g, T)
        if case["mask"]:
            st["mask"] = _rand(g, T) < 0.75
    elif kind == "policy":
        g = _gen(seed)
        st["offsets"], T = _sequences(case, g, case["n"])
        st["logp"] = -_randn(g, T).abs() * 1.5
        st["old"] = st["logp"] + 0.15 * _randn(g, T)
        if case["kl"]:
            st["ref"] = st["logp"] + 0.3 * _randn(g, T)
        st["adv"] = _randn(g, case["n"] if case["per_sequence"] else T)
        if case["ent"]:
            st["entropy"] = _randn(g, T).abs()
        if case["mask"]:
            st["mask"] = _rand(g, T) < 0.75
    elif kind == "ortho":
        g = _gen(seed)
        # a gradient's spectrum: a few strong directions over a floor
        c, r, n = case["count"], case["rows"], case["cols"]
        k = min(4, r, n)
        st["x"] = 1e-3 * (_randn(g, c, r, n) + 2.0 * torch.bmm(_randn(g, c, r, k),
                                                               _randn(g, c, k, n)))
    else:
        g = _gen(seed)
        st["shapes"] = _shapes(case)
        n = case["layers"] * sum(a * b for a, b in st["shapes"])
        st["p"] = 0.02 * _randn(g, n)
        st["g"] = 1e-3 * _randn(g, n)
        st["m"] = 5e-3 * _randn(g, n)
        if own:
            st["hp"] = _llmt().muon_hparams(lr=2e-3, momentum=0.95, wd=0.01, eps=EPS, steps=5,
                                            nesterov=case["nesterov"], scale=case["scale"])
    return st


# ---------------------------------------------------------------- the plain forms

def _plain_logp(x, t, temperature, want_entropy):
    """x [rows, V] fp32, t [rows] -> logp, stats, entropy: rows without a target are 0."""
    ok = (t >= 0) & (t < x.shape[1])
    x = x * f32(1.0 / temperature)
    m = x.amax(1)
    z = x - m[:, None]
    e = z.exp()
    s = e.sum(1)
    lp = z.gather(1, t.long().clamp(0, x.shape[1] - 1)[:, None])[:, 0] - s.log()
    zero = torch.zeros_like(lp)
    out = [torch.where(ok, lp, zero),
           torch.where(ok[:, None], torch.stack([m, s.log()], 1), zero[:, None])]
    if want_entropy:
        out.append(torch.where(ok, s.log() - (e * z).sum(1) / s, zero))
    return out


def _plain_logp_bwd(x, t, stats, dlogp, temperature, entropy, dentropy):
    it = f32(1.0 / temperature)
    ok = (t >= 0) & (t < x.shape[1])
    z = x * it - stats[:, :1] - stats[:, 1:]
    p = z.exp()
    d = -dlogp[:, None] * p
    at = t.long().clamp(0, x.shape[1] - 1)[:, None]
    d.scatter_(1, at, d.gather(1, at) + dlogp[:, None])
    if dentropy is not None:
        d = d - dentropy[:, None] * p * (z + entropy[:, None])
    return torch.where(ok[:, None], d * it, torch.zeros_like(d))


def _f(kind, z):
    """A preference loss and its derivative."""
    if kind == "sigmoid":
        return torch.relu(-z) + (-z.abs()).exp().log1p(), -1.0 / (1.0 + z.exp())
    if kind == "hinge":
        return torch.relu(1.0 - z), -(z < 1.0).to(z.dtype)
    return (z - 0.5) ** 2, 2.0 * z - 1.0


def _sums(d, offsets):
    """The sum of every sequence of d (64 bits)."""
    c = torch.zeros(d.shape[0] + 1, dtype=d.dtype, device=d.device)
    torch.cumsum(d, 0, out=c[1:])
    c = c[offsets.long()]
    return c[1:] - c[:-1]


def _segments(offsets, T):
    """The sequence of every token."""
    return torch.bucketize(torch.arange(T, device=offsets.device, dtype=torch.int32), offsets,
                           right=True).long() - 1


def _plain_pref(st):
    c = st["case"]
    n, T = c["n"], st["logp"].shape[0]
    seq = _segments(st["offsets"], T)
    d = st["logp"].double()
    if "ref" in st:
        d = d - st["ref"].double()
    keep = st["mask"] if "mask" in st else torch.ones(T, dtype=torch.bool, device=d.device)
    d = torch.where(keep, d, torch.zeros_like(d))
    r = _sums(d, st["offsets"])
    kept = _sums(keep.double(), st["offsets"])
    w = 1.0 / kept.clamp(min=1.0) if c["average"] else torch.ones_like(kept)
    r = r * w * f32(c["beta"])
    z = r[0::2] - r[1::2] - f32(c["margin"])
    e = f32(c["smooth"])
    fp, dp = _f(c["loss"], z)
    fm, dm = _f(c["loss"], -z)
    loss = (1.0 - e) * fp + e * fm
    dz = ((1.0 - e) * dp - e * dm) * (f32(c["beta"]) / n)
    dseq = torch.stack([dz, -dz], 1).reshape(-1) * w
    dlogp = torch.where(keep, dseq[seq], torch.zeros_like(d))
    return loss.mean().reshape(1).float(), loss.float(), r.float(), dlogp.float()


def _plain_policy(st):
    c = st["case"]
    n, T = c["n"], st["logp"].shape[0]
    seq = _segments(st["offsets"], T)
    lp = st["logp"].double()
    keep = st["mask"] if "mask" in st else torch.ones(T, dtype=torch.bool, device=lp.device)
    zero = torch.zeros_like(lp)
    if c["mean"] == "token":
        w = keep.double() / keep.sum().clamp(min=1)
    else:
        kept = _sums(keep.double(), st["offsets"])
        w = keep.double() / (kept.clamp(min=1.0)[seq] * n)
    adv = st["adv"].double()
    if c["per_sequence"]:
        adv = adv[seq]
    r = (lp - st["old"].double()).exp()
    lo, hi = 1.0 - f32(c["low"]), 1.0 + f32(c["high"])
    s1, s2 = r * adv, r.clamp(lo, hi) * adv
    clipped = s1 > s2
    pg = -torch.minimum(s1, s2)
    grad = torch.where(clipped, zero, -s1)
    loss = pg
    kl = zero
    if "ref" in st:
        d = st["ref"].double() - lp
        kl = torch.expm1(d) - d
        loss = loss + f32(c["kl"]) * kl
        grad = grad - f32(c["kl"]) * torch.expm1(d)
    out = {}
    if "entropy" in st:
        loss = loss - f32(c["ent"]) * st["entropy"].double()
        out["dentropy"] = (-f32(c["ent"]) * w).float()
    out["loss"] = (loss * w).sum().reshape(1).float()
    out["stats"] = torch.stack([(pg * w).sum(), (kl * w).sum(), (clipped * w).sum()]).float()
    out["dlogp"] = (grad * w).float()
    return out


def _plain_ns(x, steps, eps):
    """x [count, rows, cols] -> the Newton-Schulz iterate of x / |x|, in x's type."""
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2).contiguous()
    x = x / (x.flatten(1).norm(dim=1) + f32(eps))[:, None, None]
    for _ in range(steps):
        a = torch.bmm(x, x.transpose(1, 2).contiguous())
        x = NS[0] * x + torch.bmm(NS[1] * a + NS[2] * torch.bmm(a, a), x)
    return x.transpose(1, 2).contiguous() if tall else x


def _arena_views(flat, shapes, layers):
    """The matrices of a flat arena by place in the layer: views [layers, rows, cols]."""
    per, off, out = sum(a * b for a, b in shapes), 0, []
    for a, b in shapes:
        out.append(flat.view(layers, per)[:, off:off + a * b].unflatten(1, (a, b)))
        off += a * b
    return out


def _muon(p, g, m, shapes, layers, nesterov, scale, ns):
    """One update in p's type; returns the new p and m."""
    mu, lr, wd = f32(0.95), f32(2e-3), f32(0.01)
    m = mu * m + g
    u = g + mu * m if nesterov else m
    new = torch.empty_like(p)
    for pv, uv, nv in zip(*(_arena_views(t, shapes, layers) for t in (p, u, new))):
        a, b = pv.shape[1:]
        s = 0.2 * math.sqrt(max(a, b)) if scale == "rms" else math.sqrt(max(1.0, a / b))
        nv.copy_(pv * (1.0 - lr * wd) - lr * s * ns(uv))
    return new, m


# ---------------------------------------------------------------- one pass

def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_plain(st):
    c = st["case"]
    kind = c["kind"]
    if kind == "logp":
        return _plain_logp(st["logits"].float(), st["targets"], c["temperature"], c["entropy"])
    if kind == "logp_bwd":
        return _plain_logp_bwd(st["logits"].float(), st["targets"], st["stats"], st["dlogp"],
                               c["temperature"], st.get("entropy"),
                               st.get("dentropy")).to(st["logits"].dtype)
    if kind == "pref":
        return _plain_pref(st)
    if kind == "policy":
        return _plain_policy(st)
    if kind == "ortho":
        return _plain_ns(st["x"], c["steps"], EPS)
    new, m = _muon(st["p"], st["g"], st["m"], st["shapes"], c["layers"], c["nesterov"], c["scale"],
                   lambda u: _plain_ns(u, 5, EPS))
    st["p"].copy_(new)
    st["m"].copy_(m)
    return st["p"], st["m"]


def _run_own(st):
    llmt = _llmt()
    c = st["case"]
    kind = c["kind"]
    if kind == "logp":
        lp, stats, ent = llmt.token_logprobs(st["logits"], st["targets"],
                                             temperature=c["temperature"],
                                             want_entropy=c["entropy"])
        return [lp, stats, ent] if c["entropy"] else [lp, stats]
    if kind == "logp_bwd":
        return llmt.token_logprobs_bwd(st["logits"], st["targets"], st["stats"], st["dlogp"],
                                       entropy=st.get("entropy"), dentropy=st.get("dentropy"),
                                       temperature=c["temperature"])
    if kind == "pref":
        return llmt.preference_loss(st["logp"], st.get("ref"), st["offsets"], loss=c["loss"],
                                    beta=c["beta"], label_smoothing=c["smooth"],
                                    margin=c["margin"], average=c["average"], mask=st.get("mask"))
    if kind == "policy":
        r = llmt.policy_loss(st["logp"], st["old"], st["adv"], st["offsets"],
                             ref_logp=st.get("ref"), entropy=st.get("entropy"),
                             mask=st.get("mask"), clip_low=c["low"], clip_high=c["high"],
                             kl_coef=c["kl"], entropy_coef=c["ent"], mean=c["mean"],
                             per_sequence=c["per_sequence"])
        out = dict(loss=r.loss, stats=r.stats, dlogp=r.dlogp)
        if "entropy" in st:
            out["dentropy"] = r.dentropy
        return out
    if kind == "ortho":
        return llmt.orthogonalize(st["x"], steps=c["steps"], eps=EPS)
    llmt.muon_update(st["p"], st["g"], st["m"], st["shapes"], st["hp"])
    return st["p"], st["m"]


# ---------------------------------------------------------------- work

def work(case):
    kind = case["kind"]
    if kind in ("logp", "logp_bwd"):
        rows, v = case["rows"], case["V"]
        es = 4 if case["dtype"] == "f32" else 2
        used = rows - (math.ceil(case["skip"] * rows) if rows > 1 else 0)
        if kind == "logp":
            return {"bytes": used * v * es + rows * (4 + 4 + 8 + 4 * case["entropy"]),
                    "flops": used * v * (4 + 2 * case["entropy"])}
        return {"bytes": used * v * es + rows * v * es + rows * (16 + 8 * case["entropy"]),
                "flops": used * v * (4 + 3 * case["entropy"])}
    if kind == "pref":
        T = 2 * case["n"] * case["S"] * 0.65
        return {"bytes": T * (4 + 4 * case["ref"] + case["mask"] + 4) + case["n"] * 20,
                "flops": T * 4}
    if kind == "policy":
        T = case["n"] * case["S"] * 0.65
        per = 4 + 4 + 4 * (not case["per_sequence"]) + 4 * (case["kl"] > 0) + case["mask"] + 4
        return {"bytes": T * (per + 8 * (case["ent"] > 0)) + case["n"] * 8, "flops": T * 20}
    if kind == "ortho":
        mats = [(case["count"], case["rows"], case["cols"])]
        streams, steps = 2, case["steps"]
    else:
        mats = [(case["layers"], a, b) for a, b in _shapes(case)]
        streams, steps = 5, 5
    # read once and written once; the Gram matrix, the iteration on it and the product
    size = sum(c * a * b for c, a, b in mats)
    flops = sum(c * (3 * a * b * min(a, b) + 8 * steps * min(a, b) ** 3) for c, a, b in mats)
    return {"bytes": size * 4 * streams, "flops": flops}


# ---------------------------------------------------------------- in 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "logp":
        return _exact_logp(case, st)
    if kind == "logp_bwd":
        return _exact_logp_bwd(case, st)
    if kind == "pref":
        return _exact_pref(case, st)
    if kind == "policy":
        return _exact_policy(case, st)
    if kind == "ortho":
        return _exact_ns(st["x"].double(), case["steps"])
    return _exact_muon(case, st)


def _rows64(st, step):
    for i in range(0, st["logits"].shape[0], step):
        x = st["logits"][i:i + step].double() * f32(1.0 / st["case"]["temperature"])
        t = st["targets"][i:i + step].long()
        yield i, x, t, (t >= 0) & (t < x.shape[1])


def _exact_logp(case, st):
    lps, stats, ents = [], [], []
    for _, x, t, ok in _rows64(st, 256):
        logz = torch.logsumexp(x, 1)
        lp = x[torch.arange(len(t), device=x.device), t.clamp(min=0)] - logz
        lps.append(lp * ok)
        # the maximum and the logarithm of the sum above it
        m = x.max(1).values
        stats.append(torch.stack([m, logz - m], 1) * ok[:, None])
        if case["entropy"]:
            lg = x - logz[:, None]
            ents.append(-(lg * lg.exp()).sum(1) * ok)
    out = [torch.cat(lps), torch.cat(stats)]
    return out + [torch.cat(ents)] if case["entropy"] else out


def _exact_logp_bwd(case, st):
    # the gradients with respect to the scaled logits, row by row from the definition
    rows, v = st["logits"].shape
    if rows * v > 400_000_000:
        return None
    out = torch.empty(rows, v, dtype=torch.float64, device="cuda")
    for i, x, t, ok in _rows64(st, 128):
        lse = st["stats"][i:i + 128].double().sum(1)
        lg = x - lse[:, None]
        p = lg.exp()
        onehot = torch.zeros_like(p)
        onehot[torch.arange(len(t), device=x.device), t.clamp(min=0)] = 1.0
        d = st["dlogp"][i:i + 128].double()[:, None] * (onehot - p)
        if case["entropy"]:
            d -= st["dentropy"][i:i + 128].double()[:, None] * p * \
                (lg + st["entropy"][i:i + 128].double()[:, None])
        out[i:i + 128] = d * f32(1.0 / case["temperature"]) * ok[:, None]
    return out


def _exact_pref(case, st):
    off = st["offsets"].cpu().numpy()
    lp = st["logp"].double().cpu().numpy()
    rf = st["ref"].double().cpu().numpy() if "ref" in st else np.zeros_like(lp)
    keep = st["mask"].cpu().numpy() if "mask" in st else np.ones(len(lp), bool)
    n, beta, e = case["n"], f32(case["beta"]), f32(case["smooth"])

    def f(z):
        if case["loss"] == "sigmoid":
            return np.logaddexp(0.0, -z), -np.exp(-np.logaddexp(0.0, z))
        if case["loss"] == "hinge":
            return max(0.0, 1.0 - z), -1.0 if z < 1.0 else 0.0
        return (z - 0.5) ** 2, 2.0 * (z - 0.5)

    losses, rewards, grad = np.zeros(n), np.zeros(2 * n), np.zeros(len(lp))
    for i in range(n):
        spans = []
        for s in (2 * i, 2 * i + 1):
            at = np.arange(off[s], off[s + 1])
            at = at[keep[at]]
            w = 1.0 / max(1, len(at)) if case["average"] else 1.0
            rewards[s] = beta * w * math.fsum(lp[at] - rf[at])
            spans.append((at, w))
        z = rewards[2 * i] - rewards[2 * i + 1] - f32(case["margin"])
        (a, da), (b, db) = f(z), f(-z)
        losses[i] = (1.0 - e) * a + e * b
        dz = (1.0 - e) * da - e * db
        for sign, (at, w) in zip((1.0, -1.0), spans):
            grad[at] = sign * dz * beta * w / n
    t = torch.from_numpy
    return t(np.array([losses.mean()])), t(losses), t(rewards), t(grad)


def _exact_policy(case, st):
    off = st["offsets"].cpu().numpy()
    a = {k: st[k].double().cpu().numpy() for k in ("logp", "old", "ref", "adv", "entropy") if k in st}
    T, n = len(a["logp"]), case["n"]
    keep = st["mask"].cpu().numpy() if "mask" in st else np.ones(T, bool)
    seq = np.repeat(np.arange(n), np.diff(off))
    if case["mean"] == "token":
        w = keep / max(1, keep.sum())
    else:
        w = keep / (n * np.maximum(1, np.bincount(seq, keep, n)))[seq]
    adv = a["adv"][seq] if case["per_sequence"] else a["adv"]
    ratio = np.exp(a["logp"] - a["old"])
    lo, hi = 1.0 - f32(case["low"]), 1.0 + f32(case["high"])
    # the pessimistic side is the clipped one where the ratio has left the band in the
    # direction that the advantage rewards
    out_of_band = ((ratio > hi) & (adv > 0)) | ((ratio < lo) & (adv < 0))
    pg = -adv * np.where(out_of_band, np.clip(ratio, lo, hi), ratio)
    dlp = np.where(out_of_band, 0.0, -adv * ratio)
    kl = np.zeros(T)
    if "ref" in a:
        d = a["ref"] - a["logp"]
        kl = np.expm1(d) - d
        dlp = dlp - f32(case["kl"]) * np.expm1(d)
    loss = pg + f32(case["kl"]) * kl
    out = {}
    if "entropy" in a:
        loss = loss - f32(case["ent"]) * a["entropy"]
        out["dentropy"] = torch.from_numpy(-f32(case["ent"]) * w)
    out["loss"] = torch.tensor([math.fsum(loss * w)], dtype=torch.float64)
    out["stats"] = torch.tensor([math.fsum(pg * w), math.fsum(kl * w),
                                 math.fsum(out_of_band * w)], dtype=torch.float64)
    out["dlogp"] = torch.from_numpy(dlp * w)
    return out


def _exact_ns(x, steps, eps=EPS):
    """By the singular values: the iteration maps each of them and leaves the vectors."""
    a, b = x.shape[1:]
    if min(a, b) == 1:
        s = x.flatten(1).norm(dim=1)[:, None, None]
        y = x / s.clamp(min=1e-300)
        vals = s / (s + f32(eps))
        for _ in range(steps):
            vals = NS[0] * vals + NS[1] * vals ** 3 + NS[2] * vals ** 5
        return y * vals
    y = x if a <= b else x.transpose(1, 2)
    lam, vec = torch.linalg.eigh(y @ y.transpose(1, 2).contiguous())
    norm = x.flatten(1).norm(dim=1) + f32(eps)
    l = lam.clamp(min=0.0) / norm[:, None] ** 2
    gain = torch.ones_like(l)
    for _ in range(steps):  # s <- s (a + b s^2 + c s^4), s^2 = l
        q = NS[0] + NS[1] * l + NS[2] * l * l
        gain, l = gain * q, l * q * q
    proj = (vec * gain[:, None, :]) @ vec.transpose(1, 2).contiguous()
    y = (proj / norm[:, None, None]) @ y.contiguous()
    return y if a <= b else y.transpose(1, 2).contiguous()


def _exact_muon(case, st):
    p, m = _muon(st["p"].double(), st["g"].double(), st["m"].double(), st["shapes"],
                 case["layers"], case["nesterov"], case["scale"], lambda u: _exact_ns(u.contiguous(), 5))
    return p, m
