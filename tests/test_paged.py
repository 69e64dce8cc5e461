"""The paged KV cache's host side: sizes, and the refusal of every bad argument
before anything reaches a device."""
import ctypes as C

import numpy as np
import pytest

import paged_util as U


def test_pool_bytes():
    import g4run_amd as G
    for t in (G.F16, G.Q8_0, G.Q4_0):
        for hd in (64, 128, 256, 512):
            assert G.paged_pool_bytes(t, 3, hd, 48, 7) == 7 * U.page_bytes(t, 3, hd, 48)
    assert G.paged_pool_bytes(G.F16, 8, 128, 64, 1 << 20) == (1 << 20) * 8 * 64 * 256
    for bad in [(G.F32, 1, 64, 16, 1), (G.Q4_K, 1, 64, 16, 1), (G.F16, 0, 64, 16, 1), (G.F16, 1, 96, 16, 1), (G.F16, 1, 64, 8, 1),
                (G.F16, 1, 64, 24, 1), (G.F16, 1, 64, 4112, 1), (G.F16, 1, 64, 16, 0), (G.F16, 1 << 14, 512, 4096, 1)]:
        assert G.paged_pool_bytes(*bad) == 0, bad


def test_plain_twin_round_trips():
    # the layout of tests/paged_util.py: every byte of a row is used once
    rng = np.random.default_rng(0)
    for t in (U.F16, U.Q8_0, U.Q4_0):
        for hd in (64, 128, 256, 512):
            p = U.Pool(t, 2, hd, 16, 2)
            rows = rng.standard_normal((2, 2, 16, hd)).astype(np.float32)
            for pg in range(2):
                for h in range(2):
                    for s in range(16):
                        p.put(False, pg, s, h, rows[pg, h, s])
                        p.put(True, pg, s, h, -rows[pg, h, s])
            got = np.array([[[p.get(False, pg, s, h) for s in range(16)] for h in range(2)] for pg in range(2)])
            neg = np.array([[[p.get(True, pg, s, h) for s in range(16)] for h in range(2)] for pg in range(2)])
            assert np.array_equal(got, U.values(t, rows)) and np.array_equal(neg, U.values(t, -rows))


# Device pointers that are never used: every call below is refused first.
P = 0x1000


def _kv(G, **kw):
    d = dict(kv_type=G.F16, n_kv=2, hd=64, page=16, n_pages=4, k_dev=P, v_dev=P, status_dev=P)
    return G._PagedKV(**(d | kw))


def _batch(G, **kw):
    d = dict(n_seq=2, n_tok=3, q_off_dev=P, len_dev=P, table_dev=P, table_stride=2, max_len=32, n_prefix=0, prefix_dev=None)
    return G._PagedBatch(**(d | kw))


BAD_KV = [(dict(kv_type=0), "ERR_TYPE"), (dict(kv_type=12), "ERR_TYPE"), (dict(hd=32), "ERR_SHAPE"), (dict(hd=192), "ERR_SHAPE"),
          (dict(page=0), "ERR_SHAPE"), (dict(page=20), "ERR_SHAPE"), (dict(page=8192), "ERR_SHAPE"), (dict(n_kv=0), "ERR_SHAPE"),
          (dict(n_kv=1 << 20), "ERR_SHAPE"), (dict(n_pages=0), "ERR_ARG"), (dict(n_pages=1 << 31), "ERR_ARG"), (dict(k_dev=None), "ERR_ARG"),
          (dict(v_dev=None), "ERR_ARG"), (dict(k_dev=P + 8), "ERR_ARG"), (dict(status_dev=P + 2), "ERR_ARG")]
BAD_BATCH = [dict(n_seq=-1), dict(n_tok=-1), dict(n_tok=(1 << 24) + 1), dict(n_seq=1 << 22), dict(table_stride=-1), dict(max_len=-1),
             dict(max_len=(1 << 26) + 1), dict(n_prefix=-1), dict(n_prefix=(1 << 26) + 1), dict(len_dev=None), dict(table_dev=None),
             dict(len_dev=P + 1), dict(table_dev=P + 2), dict(q_off_dev=P + 3), dict(prefix_dev=P + 1)]


@pytest.fixture()
def abi():
    import g4run_amd as G
    return G, G.lib()


def _expect(G, rc, status):
    assert rc == getattr(G, status), (rc, G.lib().g4h_last_error())


def _append(L, kv, b, rope=None, n_head=2, q=P, qs=0, qo=2 * P, qos=0, k=P, ks=0, v=P, vs=0):
    return L.g4h_paged_append(C.byref(kv) if kv else None, C.byref(b) if b else None, C.byref(rope) if rope else None, n_head, q, qs, qo, qos,
                              k, ks, v, vs, None)


def _attn(L, kv, b, n_head=2, q=P, qs=0, scale=1.0, cap=0.0, window=0, out=1 << 20, os=0, ws=1 << 24, wsb=1 << 30):
    return L.g4h_paged_attn(C.byref(kv) if kv else None, C.byref(b) if b else None, n_head, q, qs, scale, cap, window, out, os, ws, wsb, None)


def test_refused_caches_and_batches(abi):
    G, L = abi
    calls = [lambda kv, b: _append(L, kv, b), lambda kv, b: _attn(L, kv, b),
             lambda kv, b: L.g4h_paged_read(C.byref(kv) if kv else None, C.byref(b) if b else None, G.F32, P, P, None)]
    for call in calls:
        _expect(G, call(None, _batch(G)), "ERR_ARG")
        _expect(G, call(_kv(G), None), "ERR_ARG")
        for kw, status in BAD_KV:
            _expect(G, call(_kv(G, **kw), _batch(G)), status)
        for kw in BAD_BATCH:
            _expect(G, call(_kv(G), _batch(G, **kw)), "ERR_ARG")


def test_refused_append(abi):
    G, L = abi
    kv, b = _kv(G), _batch(G)
    for kw in [dict(k=None), dict(v=None), dict(k=P + 2), dict(q=None), dict(qo=None), dict(ks=127), dict(vs=5), dict(qs=127), dict(qos=127),
               dict(n_head=-1), dict(q=P, qo=P, qs=128, qos=256)]:
        _expect(G, _append(L, kv, b, **kw), "ERR_ARG")
    for kw, status in [(dict(n_rot=4, base=1e4), "ERR_SHAPE"), (dict(n_rot=72, base=1e4), "ERR_SHAPE"), (dict(n_rot=-8, base=1e4), "ERR_SHAPE"),
                       (dict(n_rot=64, base=0.0), "ERR_ARG"), (dict(n_rot=64, base=float("nan")), "ERR_ARG"),
                       (dict(n_rot=64, base=float("inf")), "ERR_ARG"), (dict(n_rot=64, base=1e4, factor_dev=P + 1), "ERR_ARG")]:
        _expect(G, _append(L, kv, b, rope=G._Rope(**kw)), status)


def test_refused_read(abi):
    G, L = abi
    kv, b = C.byref(_kv(G)), C.byref(_batch(G))
    _expect(G, L.g4h_paged_read(kv, b, G.Q8_0, P, P, None), "ERR_TYPE")
    _expect(G, L.g4h_paged_read(kv, b, G.F32, None, None, None), "ERR_ARG")
    _expect(G, L.g4h_paged_read(kv, b, G.F32, P + 2, None, None), "ERR_ARG")
    _expect(G, L.g4h_paged_read(kv, b, G.F16, P + 1, None, None), "ERR_ARG")


def test_refused_attention(abi):
    G, L = abi
    kv, b = _kv(G), _batch(G, max_len=1 << 14, table_stride=1 << 10)
    for n_head in (0, -2, 3):
        _expect(G, _attn(L, kv, b, n_head=n_head), "ERR_SHAPE")
    need = L.g4h_paged_attn_workspace_bytes(C.byref(kv), C.byref(b), 2)
    assert need > 0
    for kw in [dict(q=None), dict(out=None), dict(q=P + 1), dict(qs=100), dict(os=100), dict(scale=float("nan")), dict(scale=float("inf")),
               dict(cap=-1.0), dict(cap=float("inf")), dict(window=-1), dict(ws=None), dict(ws=(1 << 24) + 8), dict(wsb=need - 1),
               dict(q=P, out=P), dict(q=P, out=P + 4 * 300), dict(n_head=1 << 24)]:
        _expect(G, _attn(L, kv, b, **kw), "ERR_ARG")
    _expect(G, _attn(L, kv, _batch(G, n_prefix=5)), "ERR_ARG")


def test_refused_scales(abi):
    G, L = abi
    kv, b = _kv(G), _batch(G)
    for kw in [dict(cap=2.0 ** -101), dict(cap=2.0 ** 101), dict(scale=2.0 ** 120), dict(scale=-2.0 ** 30, cap=2.0 ** -99), dict(cap=float("nan"))]:
        _expect(G, _attn(L, kv, b, **kw), "ERR_ARG")
    if not G._inited:
        for kw in [dict(cap=2.0 ** -100), dict(cap=2.0 ** 100), dict(scale=-2.0 ** 110), dict(scale=0.0)]:
            assert _attn(L, kv, b, **kw) == G.ERR_DEVICE


@pytest.mark.parametrize("hd,most", [(64, 128), (128, 128), (256, 128), (512, 64)])
def test_refused_head_groups(abi, hd, most):
    G, L = abi
    kv, b = _kv(G, hd=hd, n_kv=1), _batch(G)
    assert L.g4h_paged_attn_workspace_bytes(C.byref(kv), C.byref(b), most + 1) == 0
    _expect(G, _attn(L, kv, b, n_head=most + 1), "ERR_SHAPE")
    if not G._inited:
        assert _attn(L, kv, b, n_head=most) == G.ERR_DEVICE


def test_workspace_bytes(abi):
    G, L = abi
    size = lambda kv, b, h: L.g4h_paged_attn_workspace_bytes(C.byref(kv), C.byref(b), h)  # noqa: E731
    assert size(_kv(G), _batch(G, max_len=100), 2) == 0                   # one split: none
    assert size(_kv(G, hd=80), _batch(G), 2) == 0 and size(_kv(G), _batch(G), 3) == 0
    # it does not shrink with longer sequences
    last = 0
    for n in (100, 200, 1000, 5000, 1 << 20):
        now = size(_kv(G), _batch(G, max_len=n), 2)
        assert now >= last
        last = now


def test_good_arguments_reach_the_device_check(abi):
    # what the refusals above vary is accepted as it stands
    G, L = abi
    if G._inited:
        pytest.skip("would run on the device")
    kv, b = _kv(G), _batch(G)
    assert _append(L, kv, b, rope=G._Rope(n_rot=64, base=1e4)) == G.ERR_DEVICE
    assert _append(L, kv, b, n_head=0, q=None, qo=None) == G.ERR_DEVICE
    assert L.g4h_paged_read(C.byref(kv), C.byref(b), G.F16, P, None, None) == G.ERR_DEVICE
    assert _attn(L, kv, b) == G.ERR_DEVICE
    assert _attn(L, kv, _batch(G, q_off_dev=None), ws=None) == G.ERR_DEVICE


def test_python_class_refuses_a_bad_shape(abi):
    G, _ = abi
    with pytest.raises(G.G4HError):
        G.PagedKV(G.F16, 1, 80, 16, 4)
