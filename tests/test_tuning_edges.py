"""CPU: calls of the tuning operators whose refusal is all that keeps a kernel off memory
that is not there, or off other work than was asked for."""
import ctypes as C

import pytest

import llmt

A = lambda k: C.c_void_p(0x100000 * k)     # made-up addresses that nothing reads


@pytest.mark.parametrize("n", [1, 3000])   # one workgroup, and a workgroup a few sequences
@pytest.mark.parametrize("mean", [0, 1])
def test_advantages_a_sequence_are_needed_without_tokens_too(n, mean):
    """They are read for every sequence, however many tokens there are."""
    p = llmt.PolicyParams(mean, 1, 0.2, 0.2, 0.0, 0.0)
    rc = llmt.lib().llmt_policy_loss(None, None, None, None, None, None, A(1), 0, n, C.byref(p), A(2),
                                     A(3), None, None, A(4), 1 << 20, None)
    assert rc == llmt.LLMT_ERR_ARG
    assert llmt.lib().llmt_last_error().decode().startswith("llmt_policy_loss:")
