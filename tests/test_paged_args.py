"""The paged KV cache's host side: calls that look odd and are allowed, and calls
that look allowed and are refused."""
import ctypes as C

import pytest

from test_paged import P, _append, _attn, _batch, _kv, abi  # noqa: F401

EMPTY = [(0, 0), (3, 0), (0, 3)]


@pytest.mark.parametrize("n_seq,n_tok", EMPTY)
@pytest.mark.parametrize("q_off", [P, None])
@pytest.mark.parametrize("n_prefix", [0, 5, 5000])
@pytest.mark.parametrize("n_head", [2, 40])
def test_an_empty_batch_needs_no_workspace(abi, n_seq, n_tok, q_off, n_prefix, n_head):  # noqa: F811
    G, L = abi
    kv, b = _kv(G), _batch(G, n_seq=n_seq, n_tok=n_tok, q_off_dev=q_off, n_prefix=n_prefix, prefix_dev=P)
    assert L.g4h_paged_attn_workspace_bytes(C.byref(kv), C.byref(b), n_head) == 0
    if not G._inited:
        assert _attn(L, kv, b, n_head=n_head, ws=None, wsb=0) == G.ERR_DEVICE
