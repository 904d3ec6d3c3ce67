"""CPU: the tuning operators refuse bad arguments on the host, before any GPU work: through
the C ABI (made-up addresses that nothing reads) and in the Python binding."""
import ctypes as C
import math

import pytest
import torch

import llmt

ARG = llmt.LLMT_ERR_ARG
A = lambda k: C.c_void_p(0x100000 * k)     # 16-byte aligned, apart from one another


def logprobs(logits=A(1), dtype=0, ld=100, targets=A(2), rows=4, V=100, it=1.0, logp=A(3),
             stats=A(4), ent=None, ws=A(5), need=1 << 20):
    return llmt.lib().llmt_token_logprobs(logits, dtype, ld, targets, rows, V, it, logp, stats, ent,
                                          ws, need, None)


@pytest.mark.parametrize("bad", [
    dict(dtype=3), dict(dtype=-1), dict(ld=99), dict(rows=-1), dict(V=0, ld=0), dict(it=0.0),
    dict(V=2 ** 30 + 1, ld=2 ** 31), dict(ld=2 ** 41), dict(rows=2 ** 31 - 1, ld=2 ** 39),
    dict(it=-1.0), dict(it=math.inf), dict(it=math.nan), dict(logits=None), dict(targets=None),
    dict(logp=None), dict(stats=None), dict(logits=C.c_void_p(0x100002)),
    dict(logits=C.c_void_p(0x100001), dtype=1), dict(stats=C.c_void_p(0x400004)),
    dict(targets=C.c_void_p(0x200002)), dict(ent=C.c_void_p(0x700001))])
def test_logprobs_refusals(bad):
    assert logprobs(**bad) == ARG
    assert llmt.lib().llmt_last_error().decode().startswith("llmt_token_logprobs:")


def test_logprobs_of_no_rows_need_nothing():
    assert logprobs(logits=None, targets=None, logp=None, stats=None, rows=0, ws=None, need=0) == 0


def bwd(logits=A(1), dtype=0, ld=100, targets=A(2), stats=A(3), ent=None, dlogp=A(4), dent=None,
        rows=4, V=100, it=1.0, out=A(5), ldd=100):
    return llmt.lib().llmt_token_logprobs_bwd(logits, dtype, ld, targets, stats, ent, dlogp, dent,
                                              rows, V, it, out, ldd, None)


@pytest.mark.parametrize("bad", [
    dict(dtype=7), dict(ld=99), dict(ldd=99), dict(ldd=2 ** 62), dict(rows=-2), dict(it=0.0), dict(stats=None),
    dict(dlogp=None), dict(out=None), dict(dent=A(6)), dict(out=C.c_void_p(0x500002)),
    dict(dlogp=C.c_void_p(0x400002)), dict(dent=C.c_void_p(0x600002), ent=A(7)),
    # in place with another row stride, and overlaps that are not in place
    dict(out=A(1), ldd=101), dict(out=C.c_void_p(0x100000 + 4)),
    dict(out=C.c_void_p(0x100000 + 4 * 399)), dict(out=C.c_void_p(0x100000 - 4 * 399))])
def test_logprobs_bwd_refusals(bad):
    assert bwd(**bad) == ARG
    assert "llmt_token_logprobs_bwd" in llmt.lib().llmt_last_error().decode()


def pref(logp=A(1), ref=A(2), mask=None, off=A(3), T=10, n=2, params=(0, 0, 0.1, 0.0, 0.0),
         loss=A(4), losses=A(5), rewards=A(6), d=A(7)):
    p = None if params is None else C.byref(llmt.PrefParams(*params))
    return llmt.lib().llmt_preference_loss(logp, ref, mask, off, T, n, p, loss, losses, rewards, d,
                                           None)


@pytest.mark.parametrize("bad", [
    dict(logp=None), dict(off=None), dict(loss=None), dict(losses=None), dict(rewards=None),
    dict(params=None), dict(n=0), dict(n=2 ** 30), dict(T=-1), dict(params=(3, 0, 0.1, 0.0, 0.0)),
    dict(params=(-1, 0, 0.1, 0.0, 0.0)), dict(params=(0, 0, 0.0, 0.0, 0.0)),
    dict(params=(0, 0, math.nan, 0.0, 0.0)), dict(params=(0, 0, math.inf, 0.0, 0.0)),
    dict(params=(0, 0, 0.1, 0.6, 0.0)), dict(params=(0, 0, 0.1, -0.1, 0.0)),
    dict(params=(0, 0, 0.1, 0.0, math.inf)), dict(d=C.c_void_p(0x700002)),
    dict(off=C.c_void_p(0x300001))])
def test_preference_refusals(bad):
    assert pref(**bad) == ARG
    assert llmt.lib().llmt_last_error().decode().startswith("llmt_preference_loss:")


# enough tokens for a workspace
def policy(logp=A(1), old=A(2), ref=None, adv=A(3), ent=None, mask=None, off=A(4), T=50000, n=2,
           params=(0, 0, 0.2, 0.2, 0.0, 0.0), loss=A(5), stats=A(6), d=A(7), de=None, ws=A(8),
           need=1 << 20):
    p = None if params is None else C.byref(llmt.PolicyParams(*params))
    return llmt.lib().llmt_policy_loss(logp, old, ref, adv, ent, mask, off, T, n, p, loss, stats, d,
                                       de, ws, need, None)


@pytest.mark.parametrize("bad", [
    dict(logp=None), dict(adv=None), dict(off=None), dict(loss=None), dict(stats=None),
    dict(params=None), dict(n=0), dict(T=-1), dict(params=(2, 0, 0.2, 0.2, 0.0, 0.0)),
    dict(params=(0, 0, -0.1, 0.2, 0.0, 0.0)), dict(params=(0, 0, 1.1, 0.2, 0.0, 0.0)),
    dict(params=(0, 0, 0.2, -0.2, 0.0, 0.0)), dict(params=(0, 0, 0.2, math.nan, 0.0, 0.0)),
    dict(params=(0, 0, 0.2, 0.2, math.inf, 0.0)), dict(params=(0, 0, 0.2, 0.2, 0.0, math.nan)),
    dict(de=A(9)), dict(ws=None), dict(need=16), dict(ws=C.c_void_p(0x800008)),
    dict(adv=C.c_void_p(0x300002))])
def test_policy_refusals(bad):
    assert policy(**bad) == ARG
    assert llmt.lib().llmt_last_error().decode().startswith("llmt_policy_loss:")


# short sides above 16: these take a workspace
def ortho(x=A(1), sx=2000, ldx=100, out=A(2), so=2000, ldo=100, count=2, rows=20, cols=100, steps=5,
          eps=1e-7, ws=A(8), need=1 << 20):
    return llmt.lib().llmt_orthogonalize(x, sx, ldx, out, so, ldo, count, rows, cols, steps, eps, ws,
                                         need, None)


@pytest.mark.parametrize("bad", [
    dict(count=-1), dict(count=2 ** 21), dict(rows=0), dict(cols=0, ldx=0, ldo=0),
    dict(rows=65, sx=6500, so=6500), dict(ldx=99), dict(ldo=99), dict(sx=1999), dict(so=1999),
    dict(ldx=2 ** 62), dict(ldo=2 ** 60), dict(sx=2 ** 50), dict(so=-5), dict(ldx=-100),
    dict(steps=0), dict(steps=21), dict(eps=0.0), dict(eps=math.nan), dict(x=None), dict(out=None),
    dict(x=C.c_void_p(0x100002)), dict(ws=None), dict(need=100), dict(ws=C.c_void_p(0x800004)),
    dict(out=A(1), so=2001), dict(out=A(1), ldo=101, so=2100), dict(out=C.c_void_p(0x100004)),
    dict(out=C.c_void_p(0x100000 + 4 * 3999)), dict(cols=2 ** 30 + 1, ldx=2 ** 31, ldo=2 ** 31,
                                                    sx=2 ** 36, so=2 ** 36)])
def test_orthogonalize_refusals(bad):
    assert ortho(**bad) == ARG
    assert llmt.lib().llmt_last_error().decode().startswith("llmt_orthogonalize:")


def muon(p=A(1), g=A(2), m=A(3), layers=2, shapes=((8, 100), (50, 20)), nmat=None,
         params=(0.01, 0.9, 0.0, 1e-7, 5, 1, 0), ws=A(8), need=1 << 20):
    k = len(shapes)
    rows, cols = (C.c_int * k)(*(s[0] for s in shapes)), (C.c_int * k)(*(s[1] for s in shapes))
    hp = None if params is None else C.byref(llmt.MuonParams(*params))
    return llmt.lib().llmt_muon_update(p, g, m, layers, k if nmat is None else nmat, rows, cols, hp,
                                       ws, need, None)


@pytest.mark.parametrize("bad", [
    dict(p=None), dict(g=None), dict(m=None), dict(layers=0), dict(layers=2 ** 20), dict(nmat=0),
    dict(nmat=9), dict(shapes=((65, 65),)), dict(shapes=((0, 5),)), dict(params=None),
    dict(params=(math.nan, 0.9, 0.0, 1e-7, 5, 1, 0)), dict(params=(0.01, 1.0, 0.0, 1e-7, 5, 1, 0)),
    dict(params=(0.01, -0.1, 0.0, 1e-7, 5, 1, 0)), dict(params=(0.01, 0.9, math.inf, 1e-7, 5, 1, 0)),
    dict(params=(0.01, 0.9, 0.0, 0.0, 5, 1, 0)), dict(params=(0.01, 0.9, 0.0, 1e-7, 0, 1, 0)),
    dict(params=(0.01, 0.9, 0.0, 1e-7, 5, 1, 2)), dict(g=A(1)), dict(m=C.c_void_p(0x200004)),
    dict(p=C.c_void_p(0x300000 - 4 * 3599)), dict(ws=None), dict(need=64),
    dict(m=C.c_void_p(0x300002))])
def test_muon_refusals(bad):
    assert muon(**bad) == ARG
    assert llmt.lib().llmt_last_error().decode().startswith("llmt_muon_update:")


def test_context_muon_refuses_null():
    assert llmt.lib().llmt_muon(None, None) == ARG


def test_workspace_sizes():
    L = llmt.lib()
    assert L.llmt_policy_loss_workspace(-1, 2) == 0 and L.llmt_policy_loss_workspace(5, 0) == 0
    assert L.llmt_policy_loss_workspace(2 ** 31 - 1, 2 ** 29) < 2 ** 33
    assert L.llmt_token_logprobs_workspace(0, 100, 0) == 0
    assert L.llmt_orthogonalize_workspace(1, 65, 65) == 0 and L.llmt_orthogonalize_workspace(0, 4, 4) == 0
    assert L.llmt_orthogonalize_workspace(1, 17, 2048) > 0
    assert L.llmt_muon_update_workspace(1, 9, None, None) == 0


def test_the_binding_refuses_host_tensors():
    x, t = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32)
    off = torch.tensor([0, 1, 2], dtype=torch.int32)
    for call in (lambda: llmt.token_logprobs(x, t),
                 lambda: llmt.token_logprobs_bwd(x, t, x, x[:, 0]),
                 lambda: llmt.preference_loss(x[0], None, off),
                 lambda: llmt.policy_loss(x[0], None, x[0], off),
                 lambda: llmt.orthogonalize(x),
                 lambda: llmt.muon_update(x[0], x[1], x[1], [(2, 4)], llmt.muon_hparams()),
                 lambda: llmt.token_logprobs([1.0], t)):
        with pytest.raises(llmt.LlmtError, match="must be a device tensor"):
            call()
    with pytest.raises(llmt.LlmtError, match="loss must be one of"):
        llmt.preference_loss(x[0], None, off, loss="dpo")
    with pytest.raises(llmt.LlmtError, match="mean must be one of"):
        llmt.policy_loss(x[0], None, x[0], off, mean="sum")
    with pytest.raises(llmt.LlmtError, match="scale must be one of"):
        llmt.muon_hparams(scale="spectral")
