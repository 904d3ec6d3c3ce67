"""Float64 oracle of the packed attention and its gradients, with bounds of how far a kernel may be
off that multiplies `dtype` operands, accumulates in fp32 and rounds its outputs once.

u = eps / 2 of the type.  A score is a product of d terms in fp32: off by at most d 2^-24 times the
sum of its terms' magnitudes; the exponential's argument and value add a few fp32 roundings (2^-16
covers arguments up to 100).  A probability is then off by that share e and rounded (u):
  o  = sum P v:   (u + e) sum P |v| + u |o|
  dS = P (dP - delta):  (u + e) |dS| + P times the fp32 error of dP and delta
  dq, dk, dv: sums of |operand| times those, and u of the result.
The second factor of every bound is the sum of magnitudes, so cancellation costs what it may."""
import math

import torch


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def spans(q_off, k_off):
    q, k = q_off.tolist(), k_off.tolist()
    return [(q[s], q[s + 1], k[s], k[s + 1]) for s in range(len(q) - 1)]


def _scores(q, k, scale, see):
    s = q @ k.t() * scale
    mag = q.abs() @ k.abs().t() * scale
    return s.masked_fill(~see, -math.inf), float(mag.max()) if mag.numel() else 0.0


def _see(ql, kl, dev):
    return torch.ones(ql, kl, dtype=torch.bool, device=dev).tril(kl - ql)


def forward(q, k, v, q_off, k_off, scale):
    """(o, lse, bound of o, bound of lse) in float64."""
    d, u = q.shape[2], unit(q.dtype)
    G = q.shape[1] // k.shape[1]
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    bo, bl = torch.zeros_like(o), torch.zeros_like(lse)
    for q0, q1, k0, k1 in spans(q_off, k_off):
        if q1 == q0 or k1 == k0:
            continue
        see = _see(q1 - q0, k1 - k0, q.device)
        some = see.any(1)
        for h in range(q.shape[1]):
            kh, vh = k[k0:k1, h // G].double(), v[k0:k1, h // G].double()
            s, mag = _scores(q[q0:q1, h].double(), kh, scale, see)
            L = torch.logsumexp(s, 1)
            p = torch.exp(s - L.masked_fill(~some, 0.0)[:, None])
            lse[q0:q1, h] = L
            e = d * 2 ** -24 * mag + 2 ** -16
            bl[q0:q1, h] = d * 2 ** -24 * mag + 2 ** -18 + L.masked_fill(~some, 0.0).abs() * 2 ** -22
            o[q0:q1, h] = p @ vh
            bo[q0:q1, h] = (u + 2 * e) * (p @ vh.abs())
    return o, lse, bo + u * o.abs() + 2 ** -25, bl


def forward64(q, k, v, q_off, k_off, scale):
    """o alone, of float64 tensors."""
    G = q.shape[1] // k.shape[1]
    o = torch.zeros_like(q)
    for q0, q1, k0, k1 in spans(q_off, k_off):
        see = _see(q1 - q0, k1 - k0, q.device)
        for h in range(q.shape[1]):
            s = (q[q0:q1, h] @ k[k0:k1, h // G].t() * scale).masked_fill(~see, -math.inf)
            o[q0:q1, h] = torch.softmax(s, 1) @ v[k0:k1, h // G]
    return o


def backward(q, k, v, o, lse, do, q_off, k_off, scale):
    """((dq, dk, dv), their bounds) in float64 from the given o and lse."""
    d, u = q.shape[2], unit(q.dtype)
    G = q.shape[1] // k.shape[1]
    dq = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    dk, dv = (torch.zeros(k.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    bq, bk, bv = torch.zeros_like(dq), torch.zeros_like(dk), torch.zeros_like(dv)
    for q0, q1, k0, k1 in spans(q_off, k_off):
        if q1 == q0 or k1 == k0:
            continue
        see = _see(q1 - q0, k1 - k0, q.device)
        some = see.any(1)[:, None]
        for h in range(q.shape[1]):
            j = h // G
            qh, kh, vh = q[q0:q1, h].double(), k[k0:k1, j].double(), v[k0:k1, j].double()
            g, oh = do[q0:q1, h].double(), o[q0:q1, h].double()
            s, mag = _scores(qh, kh, scale, see)
            L = lse[q0:q1, h].double()[:, None].masked_fill(~some, 0.0)
            p = torch.exp(s - L)
            e = 2 * (d * 2 ** -24 * mag + 2 ** -16)
            dp, delta = g @ vh.t(), (g * oh).sum(1, keepdim=True)
            low = d * 2 ** -24 * (g.abs() @ vh.abs().t() + (g * oh).abs().sum(1, keepdim=True))
            ds = p * (dp - delta)
            es = (u + e) * ds.abs() + p * low * 2
            dq[q0:q1, h] += ds @ kh * scale
            bq[q0:q1, h] += es @ kh.abs() * scale
            dk[k0:k1, j] += ds.t() @ qh * scale
            bk[k0:k1, j] += es.t() @ qh.abs() * scale
            dv[k0:k1, j] += p.t() @ g
            bv[k0:k1, j] += (u + e) * (p.t() @ g.abs())
    # sums of many terms in fp32, the last rounding, and the type's smallest step
    tiny = 2 ** -25 if q.dtype == torch.float16 else 0.0
    bounds = [b * (1 + 2 ** -10) + u * x.abs() + tiny for b, x in ((bq, dq), (bk, dk), (bv, dv))]
    return (dq, dk, dv), bounds


def within(name, got, want, bound):
    got = got.double()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fin), f"{name}: non-finite values"
    assert torch.equal(got[~fin], want[~fin]), name
    off = (got - want).abs()[fin]
    worst = (off / (bound[fin] + 1e-300)).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3f} of the bound"
    return worst
