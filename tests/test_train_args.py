"""CPU: packed attention, embedding and AdamW over a list refuse bad arguments on the host, before
any GPU work: through the C ABI (made-up addresses that nothing reads) and in the Python binding."""
import ctypes as C
import math

import pytest
import torch

import llmt

ARG = llmt.LLMT_ERR_ARG
A = lambda k: 0x10000000 * k               # 16-byte aligned, far apart


def message():
    return llmt.lib().llmt_last_error().decode()


DIMS = dict(dtype=2, nq=4, nkv=2, head_dim=64, n=3, Tq=100, Tk=200, scale=0.1, q_offsets=A(1),
            k_offsets=A(2))


MANY = dict(Tq=9000, Tk=9000)


def heads(at, token, head):
    return llmt.Heads(at, token, head)


def packed(dims=None, ws=A(9), need=1 << 30, backward=False, lse=A(8), **views):
    d = None if dims is False else llmt.PackedDims(**{**DIMS, **(dims or {})})
    h = dict(q=heads(A(3), 256, 64), k=heads(A(4), 128, 64), v=heads(A(5), 128, 64),
             o=heads(A(6), 256, 64), dout=heads(A(10), 256, 64), dq=heads(A(11), 256, 64),
             dk=heads(A(12), 128, 64), dv=heads(A(13), 128, 64))
    h.update(views)
    h = {k: None if x is None else C.byref(x) for k, x in h.items()}
    d = None if d is None else C.byref(d)
    L = llmt.lib()
    if backward:
        return L.llmt_packed_attention_bwd(d, h["q"], h["k"], h["v"], h["o"], lse, h["dout"], h["dq"],
                                           h["dk"], h["dv"], ws, need, None)
    return L.llmt_packed_attention(d, h["q"], h["k"], h["v"], h["o"], lse, ws, need, None)


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("bad", [
    dict(dims=False), dict(dims=dict(dtype=0)), dict(dims=dict(dtype=3)), dict(dims=dict(nq=5)),
    dict(dims=dict(nkv=0)), dict(dims=dict(nq=0)), dict(dims=dict(nq=8192, nkv=1)),
    dict(dims=dict(nq=65, nkv=1)), dict(dims=dict(nq=130, nkv=2)),
    dict(dims=dict(nq=16, nkv=16, n=2 ** 19)), dict(dims=dict(nq=32, nkv=32, Tk=2 ** 24)),
    dict(dims=dict(head_dim=96)), dict(dims=dict(n=0)), dict(dims=dict(n=2 ** 25)),
    dict(dims=dict(Tq=-1)), dict(dims=dict(Tk=-1)), dict(dims=dict(Tq=2 ** 30)),
    dict(dims=dict(Tk=2 ** 30 + 1)), dict(dims=dict(scale=0.0)), dict(dims=dict(scale=-1.0)),
    dict(dims=dict(scale=math.nan)), dict(dims=dict(scale=math.inf)), dict(dims=dict(q_offsets=None)),
    dict(dims=dict(k_offsets=None)), dict(dims=dict(k_offsets=A(2) + 2)), dict(lse=None),
    dict(lse=A(8) + 2), dict(q=None), dict(k=None), dict(q=heads(None, 256, 64)),
    dict(q=heads(A(3) + 8, 256, 64)), dict(k=heads(A(4), 132, 64)), dict(v=heads(A(5), 128, 60)),
    dict(k=heads(A(4), 56, 64)), dict(k=heads(A(4), 2 ** 23 + 8, 64)), dict(k=heads(A(4), 128, -64)),
    dict(q=heads(A(3), 256, 2 ** 29)), dict(k=heads(A(4), 0, 64))])
def test_packed_attention_refusals(bad, backward):
    assert packed(backward=backward, **bad) == ARG
    assert message().startswith("llmt_packed_attention")


@pytest.mark.parametrize("backward,bad", [
    (False, dict(o=heads(A(6), 256, 0))), (False, dict(o=heads(A(6), 192, 64))),
    (False, dict(o=heads(A(6), 64, 64 * 99))), (False, dict(o=heads(A(3), 256, 64))),
    (False, dict(o=heads(A(3) + 128 * 100, 256, 64))), (False, dict(o=heads(A(4) - 1600, 256, 64))),
    (False, dict(o=None)), (True, dict(dq=None)), (True, dict(dout=None)), (True, dict(dk=heads(A(12), 64, 64))),
    (True, dict(dk=heads(A(13), 128, 64))), (True, dict(dq=heads(A(10), 256, 64))),
    (True, dict(dv=heads(A(5) + 256 * 199, 128, 64))), (True, dict(dims=MANY, ws=None)), (True, dict(dims=MANY, need=100)),
    (True, dict(dims=MANY, ws=A(9) + 8)), (False, dict(dims=dict(Tq=3, Tk=5000), ws=None)),
    # parts of one row that overlap by a head
    (True, dict(dq=heads(A(14), 512, 64), dk=heads(A(14) + 3 * 128, 512, 64))),
    (True, dict(dq=heads(A(14), 512, 64), dk=heads(A(14) + 4 * 128, 504, 64)))])
def test_packed_attention_output_refusals(backward, bad):
    assert packed(backward=backward, **bad) == ARG
    assert message().startswith("llmt_packed_attention")


def test_the_bindings_bytes_are_the_structs():
    assert llmt._HEADS.size == C.sizeof(llmt.Heads) and llmt._PACKED.size == C.sizeof(llmt.PackedDims)
    a = llmt.PackedDims(1, 2, 3, 4, 5, 6, 7, 0.5, 8, 9)
    assert bytes(a) == llmt._PACKED.pack(1, 2, 3, 4, 5, 6, 7, 0.5, 8, 9)
    assert bytes(llmt.Heads(1, 2, 3)) == llmt._HEADS.pack(1, 2, 3)


def test_workspaces_of_bad_sizes_are_none():
    L = llmt.lib()
    for bad in (dict(head_dim=32), dict(Tq=-1), dict(nq=3)):
        d = C.byref(llmt.PackedDims(**{**DIMS, **bad}))
        assert L.llmt_packed_attention_workspace(d) == 0 == L.llmt_packed_attention_bwd_workspace(d)
    assert L.llmt_packed_attention_workspace(None) == 0
    assert L.llmt_embedding_bwd_workspace(0, 5, 5) == 0 == L.llmt_embedding_bwd_workspace(5, 0, 5)


def embed(backward=False, tok=A(1), T=2000, w=A(2), wt=0, ldw=64, V=50, H=64, scale=1.0, x=A(3), xt=0,
          ldx=64, ws=A(4), need=1 << 30):
    L = llmt.lib()
    if backward:
        return L.llmt_embedding_bwd(tok, T, x, xt, ldx, scale, w, wt, ldw, V, H, 0, ws, need, None)
    return L.llmt_embedding(tok, T, w, wt, ldw, V, H, scale, x, xt, ldx, None)


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("bad", [
    dict(T=-1), dict(T=2 ** 23 + 1), dict(V=0), dict(V=2 ** 30 + 1, ldw=64), dict(H=0),
    dict(H=2 ** 20 + 1, ldw=2 ** 31, ldx=2 ** 31), dict(wt=3), dict(xt=-1), dict(ldw=63), dict(ldx=63),
    dict(ldw=2 ** 41), dict(ldx=2 ** 41), dict(scale=math.nan), dict(scale=math.inf), dict(tok=None),
    dict(w=None), dict(x=None), dict(w=A(2) + 2), dict(x=A(3) + 1, xt=1), dict(tok=A(1) + 2),
    dict(x=A(2)), dict(x=A(2) + 50 * 256 - 4), dict(x=A(2) - 2000 * 256 + 4)])
def test_embedding_refusals(bad, backward):
    assert embed(backward, **bad) == ARG
    assert message().startswith("llmt_embedding_bwd:" if backward else "llmt_embedding:")


@pytest.mark.parametrize("bad", [dict(ws=None), dict(need=64), dict(ws=A(4) + 4)])
def test_embedding_workspace_refusals(bad):
    assert embed(True, **bad) == ARG and "workspace" in message()


def adam(tensors=None, count=None, bits=32, hp=(1e-3, 0.9, 0.99, 1e-8, 0.0), step=1, scale=None, **bad):
    one = dict(p=A(1), g=A(2), m=A(3), v=A(4), m_exp=A(5), v_exp=A(6), copy=A(7), n=1000, g_dtype=2,
               copy_dtype=2)
    ts = [{**one, **bad}] if tensors is None else tensors
    table = (llmt.AdamTensor * len(ts))(*(llmt.AdamTensor(**t) for t in ts))
    h = None if hp is None else llmt.HParams(*hp)
    return llmt.lib().llmt_adamw_update(table, len(ts) if count is None else count, bits, h, step,
                                        scale, 0, None)


@pytest.mark.parametrize("bad", [
    dict(bits=16), dict(bits=0), dict(hp=None), dict(step=0), dict(step=-3), dict(count=-1),
    dict(count=2 ** 21), dict(hp=(math.nan, 0.9, 0.99, 1e-8, 0)), dict(hp=(1, 1.0, 0.99, 1e-8, 0)),
    dict(hp=(1, 0.9, 1.0, 1e-8, 0)), dict(hp=(1, -0.1, 0.9, 1e-8, 0)), dict(hp=(1, 0.9, 0.9, 0.0, 0)), dict(hp=(1, 0.9, 0.9, 1e-40, 0)),
    dict(hp=(1, 0.9, 0.9, 1e-8, math.inf)), dict(scale=A(8) + 2), dict(n=-1), dict(n=2 ** 41),
    dict(g_dtype=3), dict(copy_dtype=0), dict(p=None), dict(g=None), dict(m=None), dict(v=None),
    dict(bits=8, m_exp=None), dict(bits=8, v_exp=None), dict(p=A(1) + 2), dict(g=A(2) + 1),
    dict(m=A(3) + 1), dict(copy=A(7) + 1),
    # written arrays that meet
    dict(m=A(1)), dict(v=A(3) + 3996), dict(copy=A(4) + 2000), dict(g=A(1)), dict(bits=8, m_exp=A(5), v_exp=A(5) + 3),
    dict(bits=8, v=A(3) + 999)])
def test_adamw_refusals(bad):
    assert adam(**bad) == ARG
    assert message().startswith("llmt_adamw_update:")


def tensor(k, **more):
    at = lambda i: A(20 + i) + k * 0x10000
    return {**dict(p=at(0), g=at(1), m=at(2), v=at(3), m_exp=at(4), v_exp=at(5), copy=at(6), n=1000,
                   g_dtype=2, copy_dtype=2), **more}


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_refuses_the_same_tensor_twice(bits):
    """In order, out of order, and by one array alone."""
    a, b = tensor(1), tensor(2)
    for ts in ([a, a], [b, a, b], [b, tensor(0, v=a["v"]), a], [a, {**b, "copy": a["copy"] + 1998}],
               [a, {**b, "g": a["p"]}], [{**a, "p": b["v"] + 4}, b]):
        assert adam(ts, bits=bits) == ARG and "overlaps" in message()


def test_moments_refusals():
    L = llmt.lib()
    call = lambda m=A(1), v=A(2), me=A(3), ve=A(4), n=300, x=A(5), y=A(6): L.llmt_adamw_moments(
        m, v, me, ve, n, x, y, None)
    for bad in (dict(n=-1), dict(m=None), dict(v=None), dict(me=None), dict(ve=None), dict(x=None),
                dict(y=None), dict(x=A(5) + 2)):
        assert call(**bad) == ARG and message().startswith("llmt_adamw_moments:")
    assert call(n=0, m=None, v=None, me=None, ve=None, x=None, y=None) == 0


def test_no_tensors_and_no_tokens_need_nothing():
    assert adam([]) == 0
    assert adam([tensor(0, n=0, p=None, g=None, m=None, v=None)]) == 0
    assert embed(T=0, tok=None, x=None) == 0
    d = dict(dims=dict(Tq=0, Tk=0))
    none = heads(None, 0, 0)
    assert packed(**d, lse=None, q=none, k=none, v=none, o=none, ws=None, need=0) == 0


def test_the_binding_refuses_host_tensors():
    t = torch.zeros(4, dtype=torch.int32)
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: llmt.packed_attention(x, x, x, t), lambda: llmt.embedding(t, x[0]),
                 lambda: llmt.embedding_bwd(t, x[0], x[0]),
                 lambda: llmt.AdamTensors([x[0].float()], [x[0]], [llmt.adamw_state(x[0])])):
        with pytest.raises(llmt.LlmtError, match="must be a device tensor"):
            call()
    for out in ((x, x), (x, None, x)):
        with pytest.raises(llmt.LlmtError, match="three tensors"):
            llmt.packed_attention_bwd(x, x, x, x, x, x, t, out=out)
    for scale in (1e39, -1e39, "1"):
        with pytest.raises(llmt.LlmtError):
            llmt.packed_attention(x, x, x, t, scale=scale)
    with pytest.raises(llmt.LlmtError, match="32 or 8"):
        llmt.adamw_state(x, 16)
    with pytest.raises(llmt.LlmtError, match="grads"):
        llmt.AdamTensors([x], [], [llmt.adamw_state(x)])
