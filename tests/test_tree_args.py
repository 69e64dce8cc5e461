"""The refusals of the entry points over draft trees and beams: every bad argument is
refused before anything reaches a device."""
import ctypes as C

import numpy as np
import pytest

from test_paged import BAD_BATCH, BAD_KV, P, _batch, _kv, abi  # noqa: F401
from tree_util import ancestry, pack, select, walk

A = [P + 0x100000 * i for i in range(12)]                    # arrays apart from each other


def _tree(G, words=1, mask_dev=A[1], depth_dev=A[2]):
    return G._PagedTree(words, mask_dev, depth_dev)


def _attn(L, kv, b, t, n_head=2, q=A[3], qs=0, scale=1.0, cap=0.0, window=0, out=A[4], os=0, ws=A[5], wsb=1 << 40):
    r = lambda x: C.byref(x) if x is not None else None  # noqa: E731
    return L.g4h_paged_attn_tree(r(kv), r(b), r(t), n_head, q, qs, scale, cap, window, out, os, ws, wsb, None)


def _append(L, kv, b, t, rope=None, n_head=2, q=A[3], qs=0, qo=A[4], qos=0, k=A[6], ks=0, v=A[7], vs=0):
    r = lambda x: C.byref(x) if x is not None else None  # noqa: E731
    return L.g4h_paged_append_tree(r(kv), r(b), r(t), rope, n_head, q, qs, qo, qos, k, ks, v, vs, None)


def _refused(calls, status):
    for i, f in enumerate(calls):
        assert f() == status, i


def test_attention_and_append(abi):  # noqa: F811
    G, L = abi
    kv, b, t = _kv(G), _batch(G), _tree(G)
    for bad, why in BAD_KV:
        assert _attn(L, _kv(G, **bad), b, t) == getattr(G, why) and _append(L, _kv(G, **bad), b, t) == getattr(G, why), bad
    for bad in BAD_BATCH:
        assert _attn(L, kv, _batch(G, **bad), t) == G.ERR_ARG and _append(L, kv, _batch(G, **bad), t) == G.ERR_ARG, bad
    for bad in [dict(words=0), dict(words=-1), dict(words=33), dict(depth_dev=None), dict(depth_dev=P + 1), dict(mask_dev=P + 2)]:
        assert _attn(L, kv, b, _tree(G, **bad)) == G.ERR_ARG and _append(L, kv, b, _tree(G, **bad)) == G.ERR_ARG, bad
    _refused([lambda: _attn(L, kv, b, _tree(G, mask_dev=None)), lambda: _attn(L, None, b, t), lambda: _attn(L, kv, None, t), lambda: _attn(L, kv, b, None),
              lambda: _append(L, kv, b, None), lambda: _attn(L, kv, b, t, q=None), lambda: _attn(L, kv, b, t, out=None), lambda: _attn(L, kv, b, t, q=P + 1),
              lambda: _attn(L, kv, b, t, window=-1), lambda: _attn(L, kv, b, t, cap=-1.0), lambda: _attn(L, kv, b, t, scale=float("inf")),
              lambda: _attn(L, kv, b, t, qs=127), lambda: _attn(L, kv, b, t, out=A[3]),
              lambda: _attn(L, kv, _batch(G, n_prefix=5), t), lambda: _append(L, kv, b, t, k=None), lambda: _append(L, kv, b, t, qo=A[6])], G.ERR_ARG)
    assert _attn(L, kv, b, t, n_head=3) == G.ERR_SHAPE and _attn(L, kv, b, t, n_head=2 * 129) == G.ERR_SHAPE
    if not G._inited:
        assert _attn(L, kv, b, t) == G.ERR_DEVICE and _append(L, kv, b, _tree(G, mask_dev=None)) == G.ERR_DEVICE
    need = L.g4h_paged_attn_tree_workspace_bytes
    big = _batch(G, n_seq=2, n_tok=40, max_len=4000, table_stride=250)
    n = need(C.byref(kv), C.byref(big), 2)
    assert n > 0 and _attn(L, kv, big, t, ws=A[5] + 8) == G.ERR_ARG and _attn(L, kv, big, t, wsb=n - 1) == G.ERR_ARG and _attn(L, kv, big, t, ws=None) == G.ERR_ARG
    assert need(C.byref(kv), C.byref(big), 3) == 0 and need(None, C.byref(big), 2) == 0


def test_outputs_apart_from_masks_and_depths(abi):  # noqa: F811
    G, L = abi
    kv, big = _kv(G), _batch(G, n_seq=2, n_tok=40, max_len=4000, table_stride=250)
    n = L.g4h_paged_attn_tree_workspace_bytes(C.byref(kv), C.byref(big), 2)
    row = 2 * kv.hd
    for t in (_tree(G, mask_dev=A[4]), _tree(G, depth_dev=A[4]), _tree(G, mask_dev=A[4] + 40 * row * 4 - 4), _tree(G, depth_dev=A[4] - 4 * 39),
              _tree(G, mask_dev=A[5] + n - 4), _tree(G, words=3, mask_dev=A[5] - 4 * 3 * 40 + 4), _tree(G, depth_dev=A[5])):
        assert _attn(L, kv, big, t, wsb=n) == G.ERR_ARG
    # a wider stride reaches further; right behind and right before is apart
    assert _attn(L, kv, big, _tree(G, mask_dev=A[4] + 40 * row * 4), os=row + 8, wsb=n) == G.ERR_ARG
    assert _append(L, kv, big, _tree(G, depth_dev=A[4] + 40 * row * 4 - 4)) == G.ERR_ARG
    if not G._inited:
        assert _attn(L, kv, big, _tree(G, mask_dev=A[4] + 40 * row * 4, depth_dev=A[4] - 4 * 40), wsb=n) == G.ERR_DEVICE
        assert _append(L, kv, big, _tree(G, depth_dev=A[4] + 40 * row * 4)) == G.ERR_DEVICE


@pytest.mark.parametrize("n_seq,n_tok", [(0, 0), (3, 0), (0, 3)])
def test_an_empty_batch(abi, n_seq, n_tok):  # noqa: F811
    G, L = abi
    kv = _kv(G)
    b = _batch(G, n_seq=n_seq, n_tok=n_tok, q_off_dev=None, len_dev=None, table_dev=None)
    t, r = _tree(G, mask_dev=None, depth_dev=None), C.byref
    calls = [lambda: _attn(L, kv, b, t, q=None, out=None, ws=None, wsb=0), lambda: _append(L, kv, b, t, q=None, qo=None, k=None, v=None),
             lambda: L.g4h_paged_tree_build(r(b), None, 1, None, None, None, None), lambda: L.g4h_paged_keep(r(kv), 1, r(b), None, None, 1, None)]
    _refused(calls, G.OK if G._inited else G.ERR_DEVICE)


def test_build(abi):  # noqa: F811
    G, L = abi
    b = _batch(G, n_tok=100)

    def call(b=b, parent=A[1], words=2, mask=A[2], depth=A[3], status=None):
        return L.g4h_paged_tree_build(C.byref(b) if b else None, parent, words, mask, depth, status, None)

    _refused([lambda: call(b=None), lambda: call(parent=None), lambda: call(words=0), lambda: call(words=33), lambda: call(mask=None),
              lambda: call(depth=None), lambda: call(parent=P + 1), lambda: call(mask=P + 2), lambda: call(depth=P + 3), lambda: call(status=P + 2),
              lambda: call(depth=A[2] + 799 - 3), lambda: call(depth=A[1] - 396), lambda: call(mask=A[1] + 396), lambda: call(mask=P), lambda: call(depth=P + 8),
              lambda: call(b=_batch(G, n_seq=-1)), lambda: call(b=_batch(G, n_tok=-1)), lambda: call(b=_batch(G, n_tok=(1 << 24) + 1)),
              lambda: call(b=_batch(G, n_seq=(1 << 22) + 1)), lambda: call(b=_batch(G, q_off_dev=P + 1))], G.ERR_ARG)
    if not G._inited:
        assert call() == G.ERR_DEVICE and call(depth=A[2] + 800) == G.ERR_DEVICE
        assert call(b=_batch(G, n_tok=100, len_dev=None, table_dev=None, table_stride=0)) == G.ERR_DEVICE


def test_accept(abi):  # noqa: F811
    G, L = abi
    b = _batch(G, n_tok=100)

    def call(b=b, parent=A[1], token=A[2], choice=A[3], most=4, n_keep=A[4], keep=A[5], nxt=A[6], out=A[7], status=None):
        return L.g4h_paged_tree_accept(C.byref(b) if b else None, parent, token, choice, most, n_keep, keep, nxt, out, status, None)

    _refused([lambda: call(b=None), lambda: call(parent=None), lambda: call(token=None), lambda: call(choice=None), lambda: call(most=0),
              lambda: call(most=1025), lambda: call(n_keep=None), lambda: call(keep=None), lambda: call(token=P + 1), lambda: call(nxt=P + 2),
              lambda: call(out=P + 1), lambda: call(status=P + 1), lambda: call(out=P), lambda: call(out=A[5] + 28), lambda: call(nxt=A[4]),
              lambda: call(keep=A[1] + 396), lambda: call(n_keep=A[3]), lambda: call(b=_batch(G, len_dev=None)),
              lambda: call(b=_batch(G, max_len=-1))], G.ERR_ARG)
    if not G._inited:
        assert call() == G.ERR_DEVICE and call(nxt=None, out=None) == G.ERR_DEVICE


def test_keep(abi):  # noqa: F811
    G, L = abi

    def call(n=2, b=_batch(G), n_keep=A[1], keep=A[2], most=3, kv=None, **second):
        kvs = (G._PagedKV * 2)(_kv(G), _kv(G, k_dev=A[8], v_dev=A[9], **second))
        return L.g4h_paged_keep(kv or kvs, n, C.byref(b) if b else None, n_keep, keep, most, None)

    _refused([lambda: call(n=0), lambda: call(n=-1), lambda: call(n=65537), lambda: call(b=None), lambda: call(n_keep=None), lambda: call(keep=None), lambda: call(most=0),
              lambda: call(n_keep=P + 1), lambda: call(keep=P + 2)], G.ERR_ARG)
    for more in [dict(hd=128), dict(page=32), dict(n_kv=1), dict(n_pages=5), dict(kv_type=G.Q8_0)]:
        assert call(**more) == G.ERR_SHAPE, more
    assert call(hd=96) == G.ERR_SHAPE and call(kv_type=G.Q4_K) == G.ERR_TYPE
    assert L.g4h_paged_keep(None, 1, C.byref(_batch(G)), A[1], A[2], 3, None) == G.ERR_ARG
    for bad in BAD_BATCH:
        assert call(b=_batch(G, **bad)) == G.ERR_ARG, bad
    if not G._inited:
        assert call() == G.ERR_DEVICE


def test_keep_of_caches_that_share_memory(abi):  # noqa: F811
    """Rows moved in one place by two at once: refused, but where nothing is moved."""
    G, L = abi
    size = G.paged_pool_bytes(G.F16, 2, 64, 16, 4)
    far = lambda i: 1 << 32 | i << 20  # noqa: E731
    pools = [(far(2 * i), far(2 * i + 1)) for i in range(300)]

    def call(pools, b=_batch(G)):
        kvs = (G._PagedKV * len(pools))(*[_kv(G, k_dev=k, v_dev=v) for k, v in pools])
        return L.g4h_paged_keep(kvs, len(pools), C.byref(b), A[1], A[2], 3, None)

    apart = G.OK if G._inited else G.ERR_DEVICE
    for n in (2, 3, 64, 65, 300):
        few = pools[:n]
        for i, j in ((0, 1), (0, n - 1), (n // 2, n - 1)):
            if i == j:
                continue
            for pair in (few[i], few[i][::-1], (far(900), few[i][0]), (few[i][1], far(900)), (few[i][0] + size - 16, far(900)),
                         (far(900), few[i][1] - size + 16)):
                assert call(few[:j] + [pair] + few[j + 1:]) == G.ERR_ARG, (n, i, j)
        if not G._inited:                                    # right behind and right before is apart; any order
            assert call(few) == apart and call(few[::-1]) == apart
            assert call([(few[0][0] + size, far(900))] + few) == apart and call(few + [(far(900), few[-1][1] - size)]) == apart
    # nothing to move, and a fork, which only writes pages that nothing is read from
    assert call([pools[0], pools[0]], _batch(G, n_tok=0)) == apart
    if not G._inited:
        kvs = (G._PagedKV * 2)(_kv(G), _kv(G))
        assert L.g4h_paged_fork(kvs, 2, C.byref(_batch(G, n_tok=0, len_dev=A[6], table_dev=A[7])), 4, A[1], A[2], A[3], A[4], 2, None) == G.ERR_DEVICE


def test_fork(abi):  # noqa: F811
    G, L = abi

    def call(n=2, b=_batch(G, n_tok=0, len_dev=A[6], table_dev=A[7]), n_out=4, parent=A[1], fresh=A[2], lens=A[3], table=A[4], stride=2, **second):
        kvs = (G._PagedKV * 2)(_kv(G), _kv(G, k_dev=A[8], v_dev=A[9], **second))
        return L.g4h_paged_fork(kvs, n, C.byref(b) if b else None, n_out, parent, fresh, lens, table, stride, None)

    _refused([lambda: call(n=0), lambda: call(b=None), lambda: call(n_out=-1), lambda: call(n_out=(1 << 21) + 1), lambda: call(parent=None), lambda: call(fresh=None),
              lambda: call(lens=None), lambda: call(table=None), lambda: call(stride=-1), lambda: call(parent=P + 1), lambda: call(table=P + 2),
              lambda: call(table=A[7]), lambda: call(table=A[7] + 12), lambda: call(table=A[7] - 28), lambda: call(lens=A[6] + 4), lambda: call(lens=A[1]),
              lambda: call(table=A[2]), lambda: call(table=A[3]), lambda: call(b=_batch(G, len_dev=None)), lambda: call(b=_batch(G, n_seq=-1))], G.ERR_ARG)
    assert call(hd=128) == G.ERR_SHAPE
    if not G._inited:
        assert call() == G.ERR_DEVICE and call(lens=None, table=None) == G.ERR_DEVICE and call(n_out=0, parent=None, fresh=None) == G.ERR_DEVICE
        assert call(table=A[7] + 16) == G.ERR_DEVICE and call(table=A[7] - 32) == G.ERR_DEVICE


def test_beam_select(abi):  # noqa: F811
    G, L = abi

    def call(x=A[1], stride=0, g=2, b=4, v=100, s=A[2], ended=None, n=4, so=A[3], ro=A[4], to=A[5], ws=A[6], wsb=1 << 40):
        return L.g4h_beam_select(x, stride, g, b, v, s, ended, n, so, ro, to, ws, wsb, None)

    need = L.g4h_beam_workspace_bytes(2, 4, 100, 4)
    assert need > 0
    _refused([lambda: call(g=-1), lambda: call(b=0), lambda: call(b=65), lambda: call(n=0), lambda: call(n=65), lambda: call(v=0), lambda: call(v=(1 << 24) + 1),
              lambda: call(g=1 << 19), lambda: call(x=None), lambda: call(s=None), lambda: call(so=None), lambda: call(ro=None), lambda: call(to=None),
              lambda: call(x=P + 1), lambda: call(s=P + 2), lambda: call(ended=P + 1), lambda: call(so=P + 3), lambda: call(stride=99), lambda: call(stride=1 << 60),
              lambda: call(ws=None), lambda: call(ws=A[6] + 8), lambda: call(wsb=need - 1), lambda: call(so=A[1] + 3196), lambda: call(ro=A[2] + 28),
              lambda: call(to=A[2]), lambda: call(ro=A[3] + 28), lambda: call(to=A[6] + need - 4), lambda: call(so=A[2] + 4), lambda: call(so=A[2], n=5),
              lambda: call(ws=A[1]), lambda: call(ended=A[4])], G.ERR_ARG)
    for bad in [(-1, 4, 100, 4), (1, 0, 100, 4), (1, 65, 100, 4), (1, 4, 0, 4), (1, 4, 100, 0), (1, 4, 100, 65)]:
        assert L.g4h_beam_workspace_bytes(*bad) == 0, bad
    assert L.g4h_beam_workspace_bytes(0, 4, 100, 4) == 0
    if not G._inited:
        _refused([call, lambda: call(so=A[2]), lambda: call(so=A[1] + 3200), lambda: call(stride=150), lambda: call(wsb=need),
                  lambda: call(g=0, x=None, s=None, so=None, ro=None, to=None, ws=None, wsb=0)], G.ERR_DEVICE)


@pytest.mark.parametrize("n_beam,n_out", [(1, 1), (4, 8), (8, 8), (64, 64)])
@pytest.mark.parametrize("n_vocab", [1, 100, 2048, 2049, 4096, 4097, 20011, 32768, 50001, 100000, 131072, 131073, 262144, 1 << 24])
def test_a_workspace_serves_smaller_batches(abi, n_vocab, n_beam, n_out):  # noqa: F811
    """Requests end and the batch shrinks: what was enough for the largest is enough."""
    G, L = abi
    most = 0
    for g in [*range(1, 600), 1023, 1024, 1025, 1 << 14, (1 << 20) // n_beam]:
        need = L.g4h_beam_workspace_bytes(g, n_beam, n_vocab, n_out)
        assert need >= most, (g, need, most)
        most = need
    # and not far more than 2048 lists, or two a row (rows of up to 4096 tokens in parts of 2048), take
    assert most <= max(2 * g * n_beam, 2048) * (8 + 8 * n_out)

    def call(g, wsb):
        return L.g4h_beam_select(1 << 50, 0, g, n_beam, n_vocab, A[2], None, n_out, A[3], A[4], A[5], 1 << 52, wsb, None)

    for g in (1, 2, 3, 10, 31, 32, 33, 100, 128, 129, 255, 256, 257, 500):
        need = L.g4h_beam_workspace_bytes(g, n_beam, n_vocab, n_out)
        assert call(g, 0) == call(g, 7) == G.ERR_ARG
        if not G._inited:
            assert call(g, need) == G.ERR_DEVICE, g


def test_the_plain_model():
    sets, depth = ancestry([-1, 0, 0, 1, 3, -1])
    assert sets == [{0}, {0, 1}, {0, 2}, {0, 1, 3}, {0, 1, 3, 4}, {5}] and depth == [0, 1, 1, 2, 3, 0]
    assert pack([{0, 31}, {32, 40}], 2).tolist() == [[0x80000001, 0], [0, 0x101]] and pack([{33}], 1).tolist() == [[0]]
    assert walk([-1, 0, 0, 2, 2], [5, 1, 2, 2, 1], [2, 9, 1, 0, 7], 9) == ([0, 2, 4], 7) and walk([-1, 0], [5, 1], [1, 3], 1) == ([0], 1)
    x = np.log(np.array([[0.5, 0.25, 0.25], [0.25, 0.25, 0.5]], np.float64))
    s, r, t = select(x, [0.0, 0.0], 2, 4)
    assert r.tolist() == [[0, 1, 0, 0]] and t.tolist() == [[0, 2, 1, 2]] and np.allclose(s, np.log([[0.5, 0.5, 0.25, 0.25]]))
