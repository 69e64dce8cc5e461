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


def _rows(at, stride, row, n):
    return [(at + i * stride, at + i * stride + row) for i in range(n)]


@pytest.mark.parametrize("q_stride,out_stride", [(128, 128), (256, 256), (300, 300), (513, 513), (128, 256)])
def test_queries_and_outputs_may_be_columns_of_one_array(abi, q_stride, out_stride):  # noqa: F811
    G, L = abi
    if G._inited:
        pytest.skip("would run on the device")
    kv, base, n, row = _kv(G), 1 << 20, 5, 128
    b = _batch(G, n_tok=n)
    for shift in list(range(-700, 701, 20)) + [127, 128, 129, 172, 255, 256, 385, -127, -128, -129, 1153, 1664]:
        meet = any(x < d and c < y for x, y in _rows(0, q_stride, row, n) for c, d in _rows(shift, out_stride, row, n))
        ranges = shift < (n - 1) * q_stride + row and shift + (n - 1) * out_stride + row > 0
        rc = _attn(L, kv, b, q=base, qs=q_stride, out=base + 4 * shift, os=out_stride)
        refused = meet if q_stride == out_stride else ranges
        assert rc == (G.ERR_ARG if refused else G.ERR_DEVICE), (shift, meet)
    assert _attn(L, kv, _batch(G, n_tok=1), q=base, qs=1 << 62, out=base + 4 * 128, os=1 << 62) == G.ERR_DEVICE
    assert _attn(L, kv, b, q=base, qs=1 << 62, out=base + 4 * 128, os=1 << 62) == G.ERR_DEVICE


def test_append_refuses_rotated_queries_over_what_it_reads(abi):  # noqa: F811
    # n_head 2, n_kv 2, hd 64: rows of 128 floats each, three tokens
    G, L = abi
    kv, b, base, w = _kv(G), _batch(G), 1 << 20, 128 * 4 + 4
    at = lambda col: base + 4 * col  # noqa: E731
    fused = dict(q=at(0), qs=w, k=at(128), ks=w, v=at(256), vs=w)
    for kw in [dict(qo=at(4), qos=w), dict(qo=at(100), qos=w), dict(qo=at(255), qos=w), dict(qo=at(300), qos=w), dict(qo=at(w - 1), qos=w),
               dict(qo=at(-100), qos=w), dict(qo=at(-w - 127), qos=w), dict(qo=at(384), qos=w + 4)]:
        assert _append(L, kv, b, **(fused | kw)) == G.ERR_ARG, kw
    assert _append(L, kv, b, q=at(0), qo=at(64)) == G.ERR_ARG
    assert _append(L, kv, b, q=at(0), qo=at(10000), k=at(10000), v=at(0)) == G.ERR_ARG
    if not G._inited:
        for kw in [dict(qo=at(0), qos=w), dict(qo=at(384), qos=w), dict(qo=at(388), qos=w), dict(qo=at(388 - w), qos=w), dict(qo=at(5000), qos=0)]:
            assert _append(L, kv, b, **(fused | kw)) == G.ERR_DEVICE, kw
        assert _append(L, kv, b, n_head=0, **(fused | dict(qo=at(100)))) == G.ERR_DEVICE


@pytest.mark.parametrize("n_seq,n_tok", EMPTY)
@pytest.mark.parametrize("n_prefix", [0, 5])
def test_an_empty_batch_may_have_null_arrays(abi, n_seq, n_tok, n_prefix):  # noqa: F811
    G, L = abi
    kv, b = _kv(G), _batch(G, n_seq=n_seq, n_tok=n_tok, n_prefix=n_prefix, q_off_dev=None, len_dev=None, table_dev=None, prefix_dev=None)
    calls = [lambda: _append(L, kv, b, q=None, qo=None, k=None, v=None), lambda: _attn(L, kv, b, q=None, out=None, ws=None, wsb=0),
             lambda: L.g4h_paged_read(C.byref(kv), C.byref(b), G.F32, None, None, None)]
    if G._inited:
        assert [f() for f in calls] == [G.OK] * 3
    else:
        assert [f() for f in calls] == [G.ERR_DEVICE] * 3
    # other arguments are still looked at
    assert _append(L, kv, b, n_head=-1) == G.ERR_ARG and _attn(L, kv, b, window=-1) == G.ERR_ARG
    assert L.g4h_paged_read(C.byref(kv), C.byref(b), G.Q8_0, None, None, None) == G.ERR_TYPE
