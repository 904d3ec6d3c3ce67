"""GPU: the preference and policy losses where a token is impossible, where exponentials
leave their range, at every kernel's borders and far above its grid, against float64.

The kernels compute in fp64 and round each output once to fp32 (half a step, 2^-24 of
itself); the mean preference loss is a mean of rounded losses, one more half step."""
import ctypes as C
import math

import pytest
import torch
import torch.nn.functional as F

import llmt
from test_gpu_tuning_losses import close, f32, ragged
from test_gpu_tuning_losses import test_policy_loss as check_policy_loss

pytestmark = pytest.mark.gpu
INF = math.inf

# sequences and their longest length that take one workgroup, tiles of tokens, and a wave
# or a workgroup a sequence
SHAPES = [(3, 40), (3000, 5), (40, 700), (800, 300)]


def weights(off, keep, mean):
    """The weight of every token in the two means, in float64."""
    n = len(off) - 1
    if mean == "token":
        return keep.double() / max(1, int(keep.sum()))
    seq = torch.repeat_interleave(torch.arange(n), (off[1:] - off[:-1]).long())
    kept = torch.zeros(n, dtype=torch.double).index_add(0, seq, keep.double())
    return keep.double() / (kept.clamp(min=1)[seq] * n)


@pytest.mark.parametrize("mean", ["token", "sequence"])
@pytest.mark.parametrize("n,S", SHAPES)
def test_policy_without_an_old_one_at_impossible_tokens(dev, n, S, mean):
    """old_logp None: the ratio is 1 whatever the log-probability, -inf too; NaN stays NaN."""
    g = torch.Generator().manual_seed(n + S)
    off, T = ragged(g, n, S)
    lp, adv = -torch.rand(T, generator=g), torch.randn(T, generator=g)
    lp[torch.rand(T, generator=g) < 0.2] = -INF
    lp[T // 2] = -INF
    w = weights(off, torch.ones(T, dtype=torch.bool), mean)
    p = llmt.policy_loss(lp.to(dev), None, adv.to(dev), off.to(dev), mean=mean)
    want = -(adv.double() * w)
    close(p.loss, want.sum().reshape(1))
    close(p.stats, torch.stack([want.sum(), 0 * want[0], 0 * want[0]]))
    close(p.dlogp, want)
    lp[T // 2] = math.nan
    p = llmt.policy_loss(lp.to(dev), None, adv.to(dev), off.to(dev), mean=mean)
    assert p.loss.isnan() and p.dlogp[T // 2].isnan() and int(p.dlogp.isnan().sum()) == 1


@pytest.mark.parametrize("mean", ["token", "sequence"])
@pytest.mark.parametrize("n,S", SHAPES)
def test_policy_terms_beyond_exps_range(dev, n, S, mean):
    """A ratio or a KL that leaves fp64 counts nothing where its factor is 0, and +inf where
    it is not; a log-probability of -inf has an infinite KL from a finite reference."""
    g = torch.Generator().manual_seed(n * 3 + S)
    off, T = ragged(g, n, S)
    lp = -torch.rand(T, generator=g)
    old, ref, adv = lp.clone(), lp.clone(), torch.randn(T, generator=g)
    a, b, c = T // 5, T // 2, T - 1
    old[a], adv[a] = -2000.0, 0.0                # ratio exp(2000), advantage 0
    old[b], adv[b] = -INF, 0.0
    ref[c] = 1000.0
    ref[0] = -INF
    w = weights(off, torch.ones(T, dtype=torch.bool), mean)
    want = -(adv.double() * w)
    call = lambda **k: llmt.policy_loss(lp.to(dev), old.to(dev), adv.to(dev), off.to(dev), mean=mean, **k)
    for kl in (None, ref.to(dev)):
        p = call(ref_logp=kl, kl_coef=0.0)
        close(p.loss, want.sum().reshape(1))
        close(p.dlogp, want)
        assert p.stats[0] == p.loss and p.stats[1] == (0.0 if kl is None else INF)
    p = call(ref_logp=ref.to(dev), kl_coef=0.05)
    assert p.loss == INF and p.stats[1] == INF and p.dlogp[c] == -INF
    fine = torch.ones(T, dtype=torch.bool)
    fine[[0, c]] = False
    assert torch.equal(p.dlogp.cpu()[fine], call().dlogp.cpu()[fine])
    close(p.dlogp[0], want[0] + f32(0.05) * w[0])
    # an impossible token under a finite reference
    ref[c], ref[0] = lp[c], lp[0]
    lp[b], old[b] = -INF, -1.0
    p = call(ref_logp=ref.to(dev), kl_coef=0.05)
    assert p.loss == INF and p.stats[1] == INF and p.dlogp[b] == -INF
    fine = torch.arange(T) != b
    close(p.dlogp.cpu()[fine], want[fine])
    adv[a] = -1.0                                 # a weight: the loss has no bound there
    p = call()
    assert p.loss == INF and p.dlogp[a] == INF


@pytest.mark.parametrize("smooth", [0.0, 0.25])
@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "square"])
def test_preference_loss_of_an_impossible_answer(dev, kind, smooth):
    """A chosen or a rejected answer with a log-probability of -inf: the limits of f and f'."""
    off = torch.arange(7, dtype=torch.int32, device=dev)
    lp = torch.tensor([-INF, 0.0, 0.0, -INF, -1.0, -2.0], device=dev)
    mean, losses, rewards, d = llmt.preference_loss(lp, None, off, loss=kind, beta=0.5,
                                                    label_smoothing=smooth)
    e = smooth
    # f' at z = -inf and +inf of (1 - e) f(z) + e f(-z)
    lo, hi = {"sigmoid": (e - 1, e), "hinge": (e - 1, e), "square": (-INF, INF)}[kind]
    assert losses[0] == INF and losses[1] == (0.0 if e == 0 and kind != "square" else INF)
    assert mean == INF and rewards.tolist() == [-INF, 0.0, 0.0, -INF, -0.5, -1.0]
    want = torch.tensor([lo, -lo, hi, -hi], dtype=torch.double) * 0.5 / 3
    if kind == "square":
        assert d.tolist()[:4] == want.tolist()
    else:
        close(d[:4], want)
    assert d[4:].isfinite().all()


def test_sizes_beyond_32_bits_are_refused(dev):
    """The library takes sizes of 31 bits; a larger one would arrive as what its lower 32
    bits say (2^32 + 4 tokens as 4).  Nothing of the tensors is read or written."""
    N = 2 ** 32 + 4
    big = torch.empty(N, device=dev)
    ints = torch.empty(N + 1, dtype=torch.int32, device=dev)
    few, off = torch.zeros(4, device=dev), torch.tensor([0, 2, 4], dtype=torch.int32, device=dev)
    rows = big.view(N, 1)
    for call in (lambda: llmt.token_logprobs(rows, ints[:N]),
                 lambda: llmt.token_logprobs(big.view(1, N), off[:1]),
                 lambda: llmt.token_logprobs_bwd(big.view(1, N), off[:1], few[:2].view(1, 2), few[:1]),
                 lambda: llmt.preference_loss(big, None, off),
                 lambda: llmt.preference_loss(few, None, ints[:N + 1]),
                 lambda: llmt.policy_loss(big, None, few[:2], off, per_sequence=True),
                 lambda: llmt.policy_loss(few, None, few, ints),
                 lambda: llmt.orthogonalize(rows), lambda: llmt.orthogonalize(big.view(1, 1, N)),
                 lambda: llmt.orthogonalize(big.view(N, 1, 1)),
                 lambda: llmt.muon_update(big, big, big, [(1, 1)], llmt.muon_hparams())):
        with pytest.raises(llmt.LlmtError, match="at most 2"):
            call()


@pytest.mark.parametrize("n,S,per_seq,mean", [
    (5000, 9, True, "token"),          # more sequences than a workgroup keeps offsets of
    (10000, 5, True, "sequence"),      # waves of the grid take several sequences each
    (2500, 1400, False, "sequence"),   # workgroups do
    (2048, 7, True, "sequence"), (2049, 3, True, "token"), (8191, 1, False, "token"),
    (8193, 1, False, "sequence")])     # the borders of the single workgroup
def test_policy_loss_of_many_sequences(dev, n, S, per_seq, mean):
    check_policy_loss(dev, n, S, per_seq, True, True, True, True, mean)


@pytest.mark.parametrize("n,S", [(300_000, 1), (66_000, 550)])
def test_preference_loss_of_more_pairs_than_workgroups(dev, n, S):
    """Sequences of S tokens; the sums in float64 on the GPU."""
    g = torch.Generator(device="cuda").manual_seed(n)
    lp = -torch.rand(2 * n * S, generator=g, device=dev)
    off = torch.arange(0, 2 * n * S + 1, S, dtype=torch.int32, device=dev)
    mean, losses, rewards, d = llmt.preference_loss(lp, None, off, beta=0.1)
    r = lp.view(2 * n, S).double().sum(1) * f32(0.1)
    z = r[0::2] - r[1::2]
    close(rewards, r.cpu(), size=S)
    close(losses, F.softplus(-z).cpu(), size=S)
    close(mean, F.softplus(-z).mean().reshape(1).cpu(), size=S, steps=2)
    dz = -torch.sigmoid(-z) * f32(0.1) / n
    close(d.view(n, 2, S)[:, 0], dz[:, None].expand(n, S).cpu())
    close(d.view(n, 2, S)[:, 1], -dz[:, None].expand(n, S).cpu())


def guarded(x, fill):
    """x inside a larger buffer of `fill`: (the buffer, the view of x)."""
    pad = 97                                      # off 16 bytes, and more than a step of loads
    buf = torch.full((x.numel() + 2 * pad,), fill, dtype=x.dtype, device=x.device)
    view = buf[pad:pad + x.numel()]
    view.copy_(x)
    return buf, view


def unharmed(buf, fill, view):
    pad = (buf.numel() - view.numel()) // 2
    return bool((buf[:pad] == fill).all() and (buf[pad + view.numel():] == fill).all())


# (T, sequences): each kernel of either loss
@pytest.mark.parametrize("T,n", [(50, 4), (8001, 4), (30001, 4), (30001, 3000), (90001, 40),
                                 (90001, 300), (9001, 9000)])
def test_offsets_of_any_value_stay_in_guarded_arrays(dev, T, n):
    """Through the C ABI, every array inside a larger one: what is before and behind the
    outputs stays, what is before and behind the inputs (NaN) is not seen.  Offsets that are
    ascending but out of [0, T] work as if clamped; any others do no harm."""
    g = torch.Generator().manual_seed(T + n)
    L, ptr, f = llmt.lib(), llmt.ptr, torch.float32
    big = lambda size: torch.randn(size, generator=g).to(dev)
    inputs = [guarded(-big(T).abs(), math.nan)[1] for _ in range(2)]
    lp, ref = inputs
    adv, adv_seq = guarded(big(T), math.nan)[1], guarded(big(n), math.nan)[1]
    mask = guarded((torch.rand(T, generator=g) < 0.7).to(torch.uint8).to(dev), 1)[1]
    wild = torch.randint(-2 ** 31, 2 ** 31 - 1, (n + 1,), generator=g, dtype=torch.int64)
    near = torch.randint(-T // 8, T + T // 8, (n + 1,), generator=g)
    ascending = near.sort().values
    ascending[0], ascending[-1] = -2 ** 31, 2 ** 31 - 1

    def run(off):
        off = guarded(off.to(torch.int32).to(dev), 0)[1]
        out = []
        for kind in range(2):
            outs = [guarded(torch.zeros(k, device=dev), 7.0) for k in (1, n // 2, n, T)]
            p = llmt.PrefParams(0, kind, 0.1, 0.0, 0.0)
            llmt.check(L.llmt_preference_loss(ptr(lp), ptr(ref), ptr(mask), ptr(off), T, n // 2,
                                              C.byref(p), *(ptr(v) for _, v in outs), None))
            out += outs
        for mean in range(2):
            for per_seq in range(2):
                outs = [guarded(torch.zeros(k, device=dev), 7.0) for k in (1, 3, T)]
                need = L.llmt_policy_loss_workspace(T, n)
                room = torch.full((need + 64,), 7, dtype=torch.uint8, device=dev)
                p = llmt.PolicyParams(mean, per_seq, 0.2, 0.2, 0.1, 0.0)
                llmt.check(L.llmt_policy_loss(
                    ptr(lp), ptr(ref), ptr(ref), ptr(adv_seq if per_seq else adv), None, ptr(mask),
                    ptr(off), T, n, C.byref(p), *(ptr(v) for _, v in outs), None, ptr(room), need,
                    None))
                assert (room[need:] == 7).all()
                out += outs
        torch.cuda.synchronize()
        assert all(unharmed(buf, 7.0, v) for buf, v in out)
        return [v.clone() for _, v in out]

    got, want = run(ascending), run(ascending.clamp(0, T))
    assert all(torch.equal(a, b) and a.isfinite().all() for a, b in zip(got, want))
    run(near)
    run(wild)


@pytest.mark.parametrize("low", [-1e4, -1e30, torch.finfo(torch.float32).min])
@pytest.mark.parametrize("n,S", SHAPES)
def test_policy_of_tokens_behind_a_finite_mask(dev, n, S, low):
    """The same finite log-probability in all three policies, however low: ratio 1, KL 0."""
    g = torch.Generator().manual_seed(n + 7 * S)
    off, T = ragged(g, n, S)
    lp, adv = -torch.rand(T, generator=g), torch.randn(T, generator=g)
    lp[torch.rand(T, generator=g) < 0.3] = low
    w = weights(off, torch.ones(T, dtype=torch.bool), "token")
    x = lp.to(dev)
    p = llmt.policy_loss(x, x, adv.to(dev), off.to(dev), ref_logp=x, kl_coef=0.5)
    want = -(adv.double() * w)
    close(p.loss, want.sum().reshape(1))
    close(p.dlogp, want)
    assert p.stats[1] == 0 and p.stats[2] == 0
