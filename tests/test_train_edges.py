"""CPU: which layouts of outputs the packed attention takes and which it refuses as overlapping,
through the C ABI (made-up addresses that nothing reads; a call whose views are all right goes on to
refuse its missing workspace)."""
import random

import pytest

from test_train_args import A, heads, message, packed

# a call that needs a workspace: many queries, few keys
DIMS = dict(nq=4, nkv=2, head_dim=64, n=1, Tq=9000)


def accepted(dims, **views):
    assert packed({**DIMS, **dims}, backward=True, ws=None, need=0, **views) == -1
    assert "workspace" in message() or "overlaps" in message(), message()
    return "workspace" in message()


# (dims, dk, dv): keys' and values' gradients as parts of one buffer from A(12) on, bytes behind it
T, D = 50, 64
INTERLEAVED = [
    (dict(), (2 * 2 * D, 2 * D), (2 * D, 2 * 2 * D, 2 * D)),              # [T, nkv, 2, d]
    (dict(), (2 * D, T * 2 * D), (2 * D, 2 * D, T * 2 * D)),              # [nkv, T, 2, d]
    (dict(), (2 * 2 * D + 8, 2 * D), (2 * D, 2 * 2 * D + 8, 2 * D)),      # padded rows
    (dict(), (2 * D + 24, T * (2 * D + 24) + 8), (2 * D, 2 * D + 24, T * (2 * D + 24) + 8)),
    (dict(), (2 * 3 * D, 3 * D), (4 * D, 2 * 3 * D, 3 * D)),              # the outer of three
    (dict(), (2 * 2 * D, D), (2 * 2 * D, 2 * 2 * D, D)),                  # [T, 2, nkv, d]
    (dict(nkv=1), (2 * D, D), (2 * D, 2 * D, D)),                         # one head
    (dict(Tk=1), (D, 2 * D), (2 * D, D, 2 * D)),                          # one token
    (dict(Tk=1, nkv=1), (D, D), (2 * D, D, D)),
    (dict(nq=2), (2 * 3 * D, 3 * D), (2 * D, 2 * 3 * D, 3 * D)),
]


@pytest.mark.parametrize("dims,k,v", INTERLEAVED)
def test_gradients_between_one_another(dims, k, v):
    d = {"Tk": T, **dims}
    dk, dv = heads(A(12), *k), heads(A(12) + v[0], *v[1:])
    assert accepted(d, dk=dk, dv=dv) and accepted(d, dk=dv, dv=dk)
    for at in (2 * D - 16, 16):                # 16 bytes inside the other's elements
        assert not accepted(d, dk=dk, dv=heads(A(12) + at, *v[1:]))


def test_all_three_between_one_another():
    """[T, heads, 3, d] with as many query as KV heads."""
    d, row = dict(nq=4, nkv=4, Tk=9000), 4 * 3 * D
    at = [heads(A(40) + 2 * D * i, row, 3 * D) for i in range(3)]
    more = dict(q=heads(A(30), row, 3 * D), k=heads(A(30) + 2 * D, row, 3 * D),
                v=heads(A(30) + 4 * D, row, 3 * D), o=heads(A(50), 4 * D, D),
                dout=heads(A(60), 4 * D, D))
    assert accepted(d, dq=at[0], dk=at[1], dv=at[2], **more)
    assert not accepted(d, dq=at[0], dk=at[1], dv=at[0], **more)
    assert not accepted(d, dq=at[0], dk=at[1], dv=more["v"], **more)


def elements(p, token, head, tokens, nheads):
    return {p // 2 + t * token + h * head + 8 * i for t in range(tokens) for h in range(nheads)
            for i in range(D // 8)}


def test_what_is_accepted_is_apart():
    """Small views of random strides and places against their elements, listed (all multiples of 8)."""
    rng, taken = random.Random(3), 0
    for _ in range(20000):
        nkv, tk = rng.choice((1, 2, 3)), rng.choice((1, 2, 3, 5))
        one = [8 * rng.randint(8, 40), 8 * rng.choice((0, 8, 9, 16, 17, 24, rng.randint(8, 120)))]
        if rng.random() < 0.5:
            one.reverse()
        other = list(one)
        if rng.random() < 0.3:
            other[rng.randint(0, 1)] = 8 * rng.randint(8, 40)
        at = A(12) + 16 * rng.randint(-200, 200)
        d = dict(nq=nkv * 2, nkv=nkv, Tk=tk)
        q = {x: heads(A(i), 1 << 10, 64) for x, i in (("q", 20), ("o", 30), ("dout", 40), ("dq", 50))}
        rest = dict(k=heads(A(60), 1 << 10, 64), v=heads(A(70), 1 << 10, 64), **q)
        rc = packed({**DIMS, **d}, backward=True, ws=None, need=0, dk=heads(A(12), *one),
                    dv=heads(at, *other), **rest)
        assert rc == -1
        if "workspace" not in message():
            continue
        taken += 1
        a, b = elements(A(12), *one, tk, nkv), elements(at, *other, tk, nkv)
        assert len(a) == len(b) == tk * nkv * D // 8 and not a & b, (one, other, at - A(12), tk, nkv)
    assert taken > 2000
