"""Calls of packed sequences whose bounds leave no row and no key have nothing to do: they launch nothing and follow no address. No GPU: the
pointers are numbers."""
import pytest

import util  # noqa: F401  (puts the package on the path)
from fv_sdpa import _lib
from test_host_packed import BOTH, P, call


@pytest.mark.parametrize("name", BOTH)
@pytest.mark.parametrize("change", [
    dict(max_q=0, max_k=0),                                                       # a padded buffer whose sequences are all empty
    dict(max_q=0, k_tokens=0, k=None, v=None),                                    # rows in the buffer, no keys at all
    dict(max_q=0, max_k=0, q_start=None, k_start=None, q=None, k=None, v=None, out=None),
], ids=["padded", "no keys", "no addresses"])
def test_bounds_of_nothing(name, change):
    assert call(_lib.lib(), name, **change)[0] == 0


@pytest.mark.parametrize("change", [dict(max_k=0, q_tokens=0, q=None), dict(max_k=0, q_tokens=0, dout=None, dq=None, workspace=P)])
def test_bounds_of_nothing_backward(change):
    assert call(_lib.lib(), "fv_packed_attention_backward", **change)[0] == 0
