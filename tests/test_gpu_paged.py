"""The paged KV cache (append with rotation, read, attention) against float64."""
import numpy as np
import pytest

import paged_util as U
from paged_util import F16, F32, Q4_0, Q8_0, Case

pytestmark = pytest.mark.gpu
TYPES = [F16, Q8_0, Q4_0]
IDS = ["f16", "q8_0", "q4_0"]


# ----------------------------------------------------------------- attention
@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("n_head,n_kv", [(1, 1), (8, 4), (6, 2), (8, 1), (12, 1), (40, 2)])
def test_single_tokens(gpu, t, hd, n_head, n_kv):
    # lengths around the 16-slot units, the 32-position steps and the workgroup's 128
    Case(gpu, t, n_head, n_kv, hd, 16 if hd < 256 else 48, [1, 15, 16, 17, 33, 0, 128, 131, 300], seed=hd + n_head).check()


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("hd,n_head,n_kv,new,lens", [
    (64, 4, 2, [5, 1, 0, 40], [5, 90, 7, 41]),
    (128, 8, 2, [33, 2], [33, 200]),
    (128, 3, 1, [64, 1, 1, 1], [64, 64, 0, 1]),
    (256, 4, 4, [17, 50], [150, 50]),
    (512, 4, 1, [9, 20], [40, 20]),
])
def test_prompts(gpu, t, hd, n_head, n_kv, new, lens):
    Case(gpu, t, n_head, n_kv, hd, 32, lens, new=new, pad=3, seed=hd).check()


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("n_prefix,window", [(0, 0), (0, 50), (70, 0), (70, 90)])
def test_prompts_of_64_tokens_on_average(gpu, t, hd, n_prefix, window):
    # one kernel takes them all, single tokens and empty sequences too
    Case(gpu, t, 2, 1, hd, 16, [230, 300, 0, 60], new=[200, 1, 0, 60], pad=1, n_prefix=n_prefix, seed=hd).check(window=window, cap=30.0 if window else 0.0)


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("hd,heads", [(64, 128), (64, 127), (128, 128), (256, 128), (512, 64), (512, 33)])
@pytest.mark.parametrize("n_prefix", [0, 40])
def test_most_heads_of_one_kv_head(gpu, t, hd, heads, n_prefix):
    Case(gpu, t, heads, 1, hd, 16, [70, 1, 300], n_prefix=n_prefix, seed=heads).check()
    Case(gpu, t, heads, 1, hd, 16, [40, 3], new=[3, 1], n_prefix=n_prefix, seed=heads).check()


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("hd,n_kv,n_seq,longest", [(64, 4, 300, 500), (128, 2, 200, 900), (256, 2, 150, 600), (512, 1, 150, 400)])
def test_more_steps_than_workgroups(gpu, t, hd, n_kv, n_seq, longest):
    # shares that hold several short tiles, begin inside one, or end where one begins
    lens = np.random.default_rng(n_seq).integers(0, longest, n_seq)
    lens[::7] = np.arange(len(lens[::7])) % 40
    Case(gpu, t, n_kv, n_kv, hd, 16, [int(n) for n in lens], seed=hd).check()


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
def test_more_steps_of_prompts_than_workgroups(gpu, t, hd):
    rng = np.random.default_rng(hd)
    new = [int(n) for n in rng.integers(0, 90, 24)]
    lens = [n + int(m) for n, m in zip(new, rng.integers(0, 500, 24))]
    Case(gpu, t, 6 if hd < 512 else 4, 2, hd, 16, lens, new=new, seed=hd).check()


@pytest.mark.parametrize("t", TYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize("new", [[1, 1], [40, 30]])
def test_bad_scales_reach_only_their_readers(gpu, t, new):
    # an infinite scale of a value far below the row's largest weight: 0 x inf, as in the formula
    c = Case(gpu, t, 2, 1, 64, 16, [80, 37], new=new, spread=30.0, seed=41)
    clean, tol = c.expect(1.0, window=24)
    n = U.row_bytes(t, 64)
    where = ((0, 60), (1, 20))
    for seq, pos in where:
        at = c.page * n + (pos % 16) * 4
        c.pool.v[c.table[seq, pos // 16], at:at + 2] = np.asarray([np.inf], np.float16).view(np.uint8)
    c.kv.v.upload(c.pool.v)
    got = c.attn(1.0, window=24).astype(np.float64)
    for seq, pos in where:
        for i in range(c.new[seq]):
            own, r = c.lens[seq] - c.new[seq] + i, c.off[seq] + i
            if own - 24 < pos <= own:
                assert not np.isfinite(got[r, :, :32]).any(), (seq, i)
                assert np.all(np.abs(got[r, :, 32:] - clean[r, :, 32:]) <= tol[r, :, 32:])
            else:
                assert np.all(np.abs(got[r] - clean[r]) <= tol[r]), (seq, i)


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("window", [1, 5, 31, 32, 100, 1000])
@pytest.mark.parametrize("new", [[1, 1, 1], [20, 7, 33]])
def test_window(gpu, t, window, new):
    c = Case(gpu, t, 4, 2, 128, 16, [150, 300, 33], new=new, seed=window)
    c.check(window=window)
    c.check(window=window, cap=20.0)


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("cap", [0.5, 5.0, 50.0])
def test_cap(gpu, t, cap):
    # spread 3: scores up to ~100 around a cap of 0.5 to 50
    Case(gpu, t, 8, 2, 64, 32, [70, 200], spread=3.0, seed=3).check(cap=cap)


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("hd,n_head,n_kv", [(64, 8, 2), (128, 4, 4), (256, 4, 2), (512, 2, 1)])
@pytest.mark.parametrize("n_prefix", [1, 31, 129, 500])
def test_prefix(gpu, t, hd, n_head, n_kv, n_prefix):
    Case(gpu, t, n_head, n_kv, hd, 16, [1, 40, 7, 0, 16], n_prefix=n_prefix, seed=n_prefix).check()


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("window", [0, 3, 60, 250])
def test_prefix_prompts_window_cap(gpu, t, window):
    Case(gpu, t, 4, 2, 128, 32, [30, 5, 2, 64], new=[30, 5, 1, 9], pad=2, n_prefix=203, seed=4).check(window=window, cap=30.0)


@pytest.mark.parametrize("n_seq", [1, 3, 9, 40])
def test_prefix_many_rows(gpu, n_seq):
    # 8, 24, 72 and 320 rows of one KV head: every tile size
    Case(gpu, F16, 8, 1, 64, 64, [3 + i % 5 for i in range(n_seq)], n_prefix=700, seed=n_seq).check()


@pytest.mark.parametrize("t", TYPES, ids=IDS)
def test_long(gpu, t):
    Case(gpu, t, 2, 1, 64, 256, [9001, 3], seed=5).check()


def test_many_sequences(gpu):
    # more than 64 sequences: offsets scanned in several steps
    n = 150
    new = [(i * 7) % 5 for i in range(n)]
    Case(gpu, F16, 2, 1, 64, 16, [v + i % 9 for i, v in enumerate(new)], new=new, pad=5, seed=6).check()


@pytest.mark.parametrize("n", [65, 4097, 4700])
def test_thousands_of_sequences(gpu, n):
    # offsets searched in two and three levels, workgroups that pass many sequences
    new = [(i * 5) % 3 for i in range(n)]
    c = Case(gpu, F16, 1, 1, 64, 16, [v + i % 17 for i, v in enumerate(new)], new=new, pad=3, seed=n)
    c.check()
    k, v, q = _append(c, gpu, 64)
    _check_append(c, gpu, k, v, q, 64)
    Case(gpu, F16, 1, 1, 64, 16, [i % 19 for i in range(n)], n_prefix=20, seed=n).check()


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("scale", [0.0, -0.2])
@pytest.mark.parametrize("new", [None, [40, 30, 1]])
def test_scales_of_any_sign(gpu, t, scale, new):
    c = Case(gpu, t, 4, 2, 64, 16, [70, 33, 5], new=new, seed=42)
    c.check(scale=scale)
    c.check(scale=scale, cap=4.0, window=20)


@pytest.mark.parametrize("spread", [1e-4, 300.0])
def test_magnitudes(gpu, spread):
    # queries and keys far from 1; one key takes all the weight at 300
    Case(gpu, F16, 4, 2, 64, 16, [40, 100], spread=spread, seed=7).check(scale=0.125)
    Case(gpu, Q8_0, 4, 2, 64, 16, [40, 100], spread=spread, seed=7).check(scale=0.125)


def test_query_rows_of_any_size(gpu):
    c = Case(gpu, F16, 4, 2, 64, 16, [40, 100], seed=8)
    c.q[0, 0] *= 1e30                    # scores overflow the halves' range but not the scaling
    c.q[0, 1] *= 1e-38
    c.q[1, 0] = 0
    c.d["q"].upload(c.q)
    got = c.attn(1e-3).astype(np.float64)
    want, tol = c.expect(1e-3)
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("n_prefix", [0, 40])
def test_non_finite_values_reach_only_their_readers(gpu, bad, n_prefix):
    # a prompt's later tokens, and positions before the window, hold them
    c = Case(gpu, F16, 4, 2, 128, 16, [80, 37], new=[40, 30], n_prefix=n_prefix, seed=9)
    clean, tol = c.expect(0.1, window=24)
    for which in (True, False):
        x = np.zeros(128, np.float32)
        x[5] = bad
        for seq, pos in ((0, 60), (1, 20)):
            c.pool.put(which, c.table[seq, pos // 16], pos % 16, 1, x)
    c.kv.k.upload(c.pool.k)
    c.kv.v.upload(c.pool.v)
    got = c.attn(0.1, window=24).astype(np.float64)
    for seq, pos in ((0, 60), (1, 20)):
        for i in range(c.new[seq]):
            own = c.lens[seq] - c.new[seq] + i
            t = c.off[seq] + i
            sees = own - 24 < pos <= own
            assert np.all(np.abs(got[t, :2] - clean[t, :2]) <= tol[t, :2])          # KV head 0 is clean
            if sees:
                assert not np.isfinite(got[t, 2:, 5]).any(), (seq, i)
            else:
                assert np.all(np.abs(got[t, 2:] - clean[t, 2:]) <= tol[t, 2:]), (seq, i)


def test_infinite_value_is_added_as_it_is(gpu):
    c = Case(gpu, F16, 2, 1, 64, 16, [9], new=[9], seed=10)
    x = np.zeros(64, np.float32)
    x[3] = np.inf
    c.pool.put(True, c.table[0, 0], 4, 0, x)
    c.kv.v.upload(c.pool.v)
    got = c.attn(0.1)
    assert np.all(np.isposinf(got[4:, :, 3])) and np.isfinite(got[:4]).all() and np.isfinite(np.delete(got, 3, 2)).all()


@pytest.mark.parametrize("t", TYPES, ids=IDS)
def test_strides(gpu, t):
    G = gpu
    c = Case(G, t, 4, 2, 64, 16, [20, 50, 3], new=[3, 1, 2], seed=11)
    want, tol = c.expect(0.125)
    for pad, shift in ((5, 1), (8, 4)):                  # unaligned rows, aligned rows
        stride = 4 * 64 + pad
        x = np.zeros(c.n_tok * stride + shift, np.float32)
        x[shift:].reshape(c.n_tok, stride)[:, :256] = c.q.reshape(c.n_tok, 256)
        q, out = G.Buffer.from_array(x), G.Buffer.from_array(np.full_like(x, 3.0))
        G.paged_attn(c.kv, c.batch, q.ptr + 4 * shift, 4, out.ptr + 4 * shift, scale=0.125, q_stride=stride, out_stride=stride)
        got = out.download(np.float32, x.shape)
        rows = got[shift:].reshape(c.n_tok, stride)
        assert np.all(np.abs(rows[:, :256].reshape(want.shape) - want) <= tol)
        assert np.all(rows[:, 256:] == 3.0) and np.all(got[:shift] == 3.0)


def test_same_page_twice_and_shared_between_sequences(gpu):
    # two sequences (and a prefix) that name the same pages read the same rows
    c = Case(gpu, F16, 2, 2, 64, 16, [32, 32], n_prefix=16, seed=12)
    c.table[1] = c.table[0]
    c.table[0, 1] = c.table[0, 0]
    c.prefix[0] = c.table[0, 0]
    c.rows[1] = [x.copy() for x in c.rows[0]]
    for w in (0, 1):
        c.rows[0][w][16:] = c.rows[0][w][:16]
        c.shared[w][:] = c.rows[0][w][:16]
    c.d["table"].upload(c.table)
    c.d["pre"].upload(c.prefix)
    c.check()


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("where", ["own", "prefix", "negative"])
def test_bad_page_is_flagged(gpu, t, where):
    c = Case(gpu, t, 2, 1, 64, 16, [60, 40, 20], n_prefix=20, seed=13)
    want, tol = c.expect(0.1)
    if where == "prefix":
        c.prefix[1] = c.pool.n_pages
        c.d["pre"].upload(c.prefix)
        hit = [0, 1, 2]
    else:
        c.table[1, 1] = -1 if where == "negative" else c.pool.n_pages + 5
        c.d["table"].upload(c.table)
        hit = [1]
    got = c.attn(0.1)
    assert c.kv.status() == gpu.PAGED_BAD_PAGE and c.kv.status() == 0
    for s in range(3):
        if s in hit:
            assert np.isnan(got[s]).all()
        else:
            assert np.all(np.abs(got[s] - want[s]) <= tol[s])


@pytest.mark.parametrize("n_prefix", [0, 20])
@pytest.mark.parametrize("value", [-1, 61, 1 << 30])
def test_bad_length_is_flagged(gpu, value, n_prefix):
    c = Case(gpu, F16, 2, 1, 64, 16, [60, 40, 20], n_prefix=n_prefix, seed=14)
    want, tol = c.expect(0.1)
    c.d["lens"].upload(np.asarray([60, value, 20, 0], np.int32))
    got = c.attn(0.1)
    assert c.kv.status() == gpu.PAGED_BAD_BATCH
    assert np.isnan(got[1]).all()
    for s in (0, 2):
        assert np.all(np.abs(got[s] - want[s]) <= tol[s])


def test_bad_offsets_are_flagged(gpu):
    c = Case(gpu, F16, 2, 1, 64, 16, [60, 40, 20], new=[2, 3, 1], seed=15)
    want, tol = c.expect(0.1)
    c.d["off"].upload(np.asarray([0, 2, 9, 6], np.int32))           # past n_tok, then descending
    got = c.attn(0.1)
    assert c.kv.status() == gpu.PAGED_BAD_BATCH
    assert np.all(np.abs(got[:2] - want[:2]) <= tol[:2])


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("n_prefix", [0, 100])
def test_graph_replays_with_other_lengths(gpu, t, n_prefix):
    """A captured call is replayed with lengths, pages and inputs changed on the
    device, eager work between the replays."""
    G = gpu
    c = Case(G, t, 4, 2, 64, 16, [130, 200, 90, 1], new=[2, 1, 3, 1], pad=1, n_prefix=n_prefix, seed=16)
    s = G.Stream()
    ws = G.Buffer(max(16, G.paged_attn_workspace_bytes(c.kv, c.batch, 4)))
    out = G.Buffer.from_array(np.full((c.n_tok, 4, 64), 7.5, np.float32))
    g = G.Graph(s.ptr, lambda: G.paged_attn(c.kv, c.batch, c.d["q"], 4, out, scale=0.125, ws=ws, stream=s.ptr))
    full = [x[:] for x in c.rows]
    for step, lens in enumerate([[130, 200, 90, 1], [5, 17, 3, 0], [129, 64, 33, 1], [130, 200, 90, 1]]):
        c.lens = lens
        c.rows = [[w[:n] for w in x] for x, n in zip(full, lens)]
        c.q = (c.rng.standard_normal(c.q.shape)).astype(np.float32)
        c.d["q"].upload(c.q, s.ptr)
        c.d["lens"].upload(np.asarray(lens + [0], np.int32), s.ptr)
        g.launch(s.ptr)
        s.synchronize()
        got = out.download(np.float32, (c.n_tok, 4, 64))
        want, tol = c.expect(0.125)
        assert np.all(np.abs(got - want) <= tol), step
        eager = c.attn(0.125)
        assert np.array_equal(eager, got), step
    assert c.kv.status() == 0


def test_two_graphs_over_one_workspace(gpu):
    """A decode call and a call of prompts, captured apart over one workspace,
    replayed one after the other; what the other left in it changes nothing."""
    G = gpu
    a = Case(G, F16, 8, 2, 128, 16, [400, 33, 0, 250], n_prefix=100, seed=18)
    b = Case(G, Q8_0, 8, 2, 64, 16, [300, 290, 7], new=[150, 30, 7], pad=2, seed=19)
    s = G.Stream()
    ws = G.Buffer(max(G.paged_attn_workspace_bytes(c.kv, c.batch, 8) for c in (a, b)))
    ws.upload(np.full(ws.nbytes, 0xff, np.uint8))
    outs = [G.Buffer.from_array(np.full((c.n_tok, 8, c.hd), 7.5, np.float32)) for c in (a, b)]
    gs = [G.Graph(s.ptr, lambda c=c, o=o: G.paged_attn(c.kv, c.batch, c.d["q"], 8, o, scale=0.1, ws=ws, stream=s.ptr)) for c, o in zip((a, b), outs)]
    want = [c.expect(0.1) for c in (a, b)]
    for turn in range(4):
        for k in ((0, 1), (1, 0))[turn & 1]:
            gs[k].launch(s.ptr)
            s.synchronize()
            got = outs[k].download(np.float32, want[k][0].shape)
            assert np.all(np.abs(got - want[k][0]) <= want[k][1]), (turn, k)


def test_streams_run_side_by_side(gpu):
    G = gpu
    cases = [Case(G, t, 4, 2, 128, 16, [300, 64], seed=17 + t) for t in TYPES]
    streams = [G.Stream() for _ in cases]
    ws = [G.Buffer(max(16, G.paged_attn_workspace_bytes(c.kv, c.batch, 4))) for c in cases]
    outs = [G.Buffer(c.n_tok * 4 * 128 * 4) for c in cases]
    for _ in range(5):
        for c, s, w, o in zip(cases, streams, ws, outs):
            G.paged_attn(c.kv, c.batch, c.d["q"], 4, o, scale=0.1, ws=w, stream=s.ptr)
    for c, s, o in zip(cases, streams, outs):
        s.synchronize()
        want, tol = c.expect(0.1)
        assert np.all(np.abs(o.download(np.float32, want.shape) - want) <= tol)


def test_runs_repeat_bit_for_bit(gpu):
    c = Case(gpu, Q8_0, 8, 2, 128, 32, [700, 33, 90], n_prefix=150, seed=20)
    first = c.attn(0.1)
    for _ in range(3):
        assert np.array_equal(c.attn(0.1), first)


def test_offsets_past_32_bits(gpu):
    """Pages more than 4 GiB into the pools."""
    G = gpu
    page, hd, n_kv = 64, 128, 8
    pb = U.page_bytes(F16, n_kv, hd, page)
    n_pages = (9 << 30) // 2 // pb
    kv = G.PagedKV(F16, n_kv, hd, page, n_pages)
    c = Case(G, F16, 16, n_kv, hd, page, [100], seed=21)
    table = np.asarray([[n_pages - 1, n_pages - 2]], np.int32)
    L = G.lib()
    for i in range(2):
        for buf, rows in ((kv.k, c.pool.k), (kv.v, c.pool.v)):
            row = np.ascontiguousarray(rows[c.table[0, i]])
            G.check(L.g4h_memcpy_h2d(buf.ptr + int(table[0, i]) * pb, row.ctypes.data, pb, None))
            G.synchronize()
    c.kv = kv
    c.d["table"].upload(table)
    c.check()
    k, v = G.Buffer(n_kv * hd * 4), G.Buffer(n_kv * hd * 4)
    G.paged_read(kv, c.batch, k, v)
    assert np.array_equal(k.download(np.float32, (n_kv, hd)), c.rows[0][0][99])
    assert np.array_equal(v.download(np.float32, (n_kv, hd)), c.rows[0][1][99])


# ------------------------------------------------------------ append and read
def _append(c, G, n_rot, base=1e4, interleaved=False, factors=None, q_out=None, fused=False, stream=None):
    k = c.rng.standard_normal((c.n_tok, c.n_kv, c.hd)).astype(np.float32)
    v = c.rng.standard_normal((c.n_tok, c.n_kv, c.hd)).astype(np.float32)
    rope = G.Rope(n_rot, base, interleaved, G.Buffer.from_array(factors) if factors is not None else None) if n_rot else None
    if fused:
        x = np.concatenate([c.q, k, v], 1).reshape(c.n_tok, -1)
        w, hd = x.shape[1], c.hd
        b = G.Buffer.from_array(x)
        G.paged_append(c.kv, c.batch, b.ptr + 4 * c.n_head * hd, b.ptr + 4 * (c.n_head + c.n_kv) * hd, q=b, q_out=b, n_head=c.n_head, rope=rope,
                       q_stride=w, q_out_stride=w, k_stride=w, v_stride=w, stream=stream)
        G.synchronize(stream)
        y = b.download(np.float32, x.shape)
        assert np.array_equal(y[:, c.n_head * hd:], x[:, c.n_head * hd:])
        return k, v, y[:, :c.n_head * hd].reshape(c.q.shape)
    kb, vb, qo = G.Buffer.from_array(k), G.Buffer.from_array(v), q_out or G.Buffer.from_array(np.full_like(c.q, 7.5))
    G.paged_append(c.kv, c.batch, kb, vb, q=c.d["q"], q_out=qo, n_head=c.n_head, rope=rope, stream=stream)
    G.synchronize(stream)
    return k, v, qo.download(np.float32, c.q.shape)


def _tokens(c):
    """(token, sequence, own position) of the tokens that have one."""
    return [(c.off[s] + i, s, n - m + i) for s, (m, n) in enumerate(zip(c.new, c.lens)) for i in range(m) if n - m + i >= 0]


def _check_append(c, G, k, v, q, n_rot, base=1e4, interleaved=False, factors=None, before=None):
    """q, the pools and the read-back against the plain twin.  A rotated element
    carries the roundings of cos and sin (the angle's fraction of a turn in fp32:
    2^-24, times 2 pi; 2^-24 of the functions), two products and a sum: 2^-21
    of the pair's size.  Stored: half a step of the type's rounding more, a whole
    one where that error crosses a border."""
    toks = _tokens(c)
    pos = np.full(c.n_tok, 0.0)
    for t, s, own in toks:
        pos[t] = c.n_prefix + own
    size = lambda x: np.abs(x).max(-1, keepdims=True) * 2 * 2.0 ** -21  # noqa: E731
    wq, wk = U.turn(c.q, pos, n_rot, base, interleaved, factors), U.turn(k, pos, n_rot, base, interleaved, factors)
    has = np.zeros(c.n_tok, bool)
    has[[t for t, _, _ in toks]] = True
    assert np.all(np.abs(q - wq)[has] <= np.broadcast_to(size(c.q), q.shape)[has])
    kb, vb = (G.Buffer.from_array(np.full((c.n_tok, c.n_kv, c.hd), 9.0, np.float32)) for _ in range(2))
    G.paged_read(c.kv, c.batch, kb, vb)
    gk, gv = (b.download(np.float32, (c.n_tok, c.n_kv, c.hd)) for b in (kb, vb))
    assert np.all(gk[~has] == 9.0) and np.all(gv[~has] == 9.0)
    assert np.array_equal(gv[has], U.values(c.t, v)[has].astype(np.float32))
    err = np.broadcast_to(size(k), k.shape)
    if c.t == F16:
        tol = np.abs(wk) * 2.0 ** -11 + 2.0 ** -25 + 2 * err
    else:
        top = np.abs(wk).reshape(*wk.shape[:-1], -1, 32).max(-1)
        step = np.repeat(top / (127 if c.t == Q8_0 else 8), 32, -1)
        # q8_0: half a step; q4_0: the value opposite the largest is cut at 7 steps
        tol = step * (0.5 if c.t == Q8_0 else 1.0) * (1 + 2.0 ** -9) + np.abs(wk) * 2.0 ** -10 + 2.0 ** -24 * 128 + 2 * err
    assert np.all(np.abs(gk - wk)[has] <= tol[has])
    # the pools hold what was read, in the layout, and nothing else changed
    pk, pv = c.kv.k.download(np.uint8, c.pool.k.shape), c.kv.v.download(np.uint8, c.pool.v.shape)
    old_k, old_v = c.pool.k, c.pool.v
    c.pool.k, c.pool.v = pk, pv
    for t, s, own in toks:
        for h in range(c.n_kv):
            at = (c.table[s, own // c.page], own % c.page, h)
            assert np.array_equal(c.pool.get(False, *at), gk[t, h].astype(np.float64))
            assert np.array_equal(c.pool.get(True, *at), gv[t, h].astype(np.float64))
    c.pool.k, c.pool.v = old_k.copy(), old_v.copy()
    for t, s, own in toks:
        for h in range(c.n_kv):
            at = (c.table[s, own // c.page], own % c.page, h)
            c.pool.put(True, *at, v[t, h])
            n, row = U.row_bytes(c.t, c.hd), h * c.page + at[1]
            c.pool.k[at[0], row * n:(row + 1) * n] = pk[at[0], row * n:(row + 1) * n]
            if c.t != F16:
                a = c.n_kv * c.page * n + row * (c.hd // 16)
                c.pool.k[at[0], a:a + c.hd // 16] = pk[at[0], a:a + c.hd // 16]
    assert np.array_equal(c.pool.v, pv) and np.array_equal(c.pool.k, pk)
    assert c.kv.status() == 0


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("hd,n_head,n_kv", [(64, 1, 1), (64, 6, 3), (128, 8, 2), (256, 8, 4), (512, 5, 1)])
@pytest.mark.parametrize("new", [None, [3, 0, 20, 1]])
def test_append(gpu, t, hd, n_head, n_kv, new):
    c = Case(gpu, t, n_head, n_kv, hd, 16, [17, 5, 33, 0], new=new, pad=0 if new is None else 2, seed=hd)
    k, v, q = _append(c, gpu, hd)
    _check_append(c, gpu, k, v, q, hd)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hd,n_rot", [(64, 0), (64, 8), (128, 64), (256, 256), (512, 128), (512, 512)])
def test_append_rotations(gpu, interleaved, hd, n_rot):
    factors = (1.0 + np.arange(n_rot // 2) % 3).astype(np.float32) if n_rot else None
    c = Case(gpu, F16, 3, 2, hd, 32, [40, 9], new=[4, 9], seed=n_rot)
    k, v, q = _append(c, gpu, n_rot, 5e5, interleaved, factors)
    _check_append(c, gpu, k, v, q, n_rot, 5e5, interleaved, factors)


def test_append_far_positions(gpu):
    # behind a prefix of 2^26 - 3 positions: the angle is taken in 64 bits
    G = gpu
    c = Case(G, F16, 2, 1, 128, 16, [20], new=[5], seed=30)
    c.n_prefix = c.batch.struct.n_prefix = (1 << 26) - 3
    k, v, q = _append(c, G, 128)
    _check_append(c, G, k, v, q, 128)


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("hd", [64, 512])
def test_append_fused_rows_in_place(gpu, t, hd):
    c = Case(gpu, t, 4, 2, hd, 16, [30, 12, 7], new=[6, 12, 1], seed=31)
    k, v, q = _append(c, gpu, hd, fused=True)
    _check_append(c, gpu, k, v, q, hd)


def test_append_many_tokens(gpu):
    # whole rows per workgroup, several tokens each
    c = Case(gpu, Q8_0, 2, 1, 64, 64, [4500, 4100], new=[4400, 4100], seed=32)
    k, v, q = _append(c, gpu, 64)
    _check_append(c, gpu, k, v, q, 64)


@pytest.mark.parametrize("t", [Q8_0, Q4_0], ids=IDS[1:])
def test_append_special_blocks(gpu, t):
    # zero blocks, ties of the largest magnitude with both signs, tiny values
    G = gpu
    c = Case(G, t, 1, 1, 128, 16, [4], new=[4], seed=33)
    v = c.rng.standard_normal((4, 1, 128)).astype(np.float32)
    v[0, 0, :32] = 0
    v[1, 0, 5], v[1, 0, 20], v[1, 0, 40], v[1, 0, 34] = 9.0, -9.0, -9.0, 9.0
    v[2] *= 1e-5
    v[3] = np.sign(v[3])
    kb, vb = G.Buffer.from_array(v), G.Buffer.from_array(v)
    G.paged_append(c.kv, c.batch, kb, vb)
    ko, vo = G.Buffer(v.nbytes), G.Buffer(v.nbytes)
    G.paged_read(c.kv, c.batch, ko, vo)
    want = U.values(t, v).astype(np.float32)
    assert np.array_equal(ko.download(np.float32, v.shape), want) and np.array_equal(vo.download(np.float32, v.shape), want)


def test_read_half(gpu):
    G = gpu
    c = Case(G, Q4_0, 1, 2, 64, 16, [20], new=[20], seed=34)
    k = G.Buffer(20 * 2 * 64 * 2)
    G.paged_read(c.kv, c.batch, k, None, out_type=F16)
    assert np.array_equal(k.download(np.float16, (20, 2, 64)), c.rows[0][0].astype(np.float16))


@pytest.mark.parametrize("t", TYPES, ids=IDS)
def test_append_bad_pages_and_lengths(gpu, t):
    G = gpu
    c = Case(G, t, 1, 1, 64, 16, [20, 20, 20, 20], seed=35)
    before_k, before_v = c.pool.k.copy(), c.pool.v.copy()
    c.table[0, 1], c.table[1, 1] = -1, c.pool.n_pages
    c.d["table"].upload(c.table)
    c.d["lens"].upload(np.asarray([20, 20, 21, 20, 0], np.int32))
    k, v, q = _append(c, G, 64)
    assert c.kv.status() == G.PAGED_BAD_PAGE | G.PAGED_BAD_BATCH
    pk, pv = c.kv.k.download(np.uint8, before_k.shape), c.kv.v.download(np.uint8, before_v.shape)
    changed = {int(i) for i in np.argwhere((pk != before_k).any(1) | (pv != before_v).any(1))[:, 0]}
    assert changed == {int(c.table[3, 1])}
    out = G.Buffer.from_array(np.full((4, 1, 64), 9.0, np.float32))
    G.paged_read(c.kv, c.batch, out, None)
    assert c.kv.status() == G.PAGED_BAD_PAGE | G.PAGED_BAD_BATCH
    assert np.all(out.download(np.float32, (4, 1, 64))[:3] == 9.0)


# ------------------------------------------------------------ together
@pytest.mark.parametrize("t", TYPES, ids=IDS)
def test_a_served_batch(gpu, t):
    """A fused projection through g4h_matmul, its rows appended and attended,
    prompt first and then token by token from a captured graph whose lengths
    advance, against the attention over the values the cache holds."""
    from g4run_amd import synth
    G = gpu
    n_head, n_kv, hd, width, n_pre, page = 4, 2, 64, 256, 50, 16
    c = Case(G, t, n_head, n_kv, hd, page, [40, 40, 40], new=[30, 7, 1], n_prefix=n_pre, seed=40)
    total = (n_head + 2 * n_kv) * hd
    W = G.Tensor.from_rows(G.Q8_0, synth.weights(G.Q8_0, total, width, seed=1), width)
    lens = [30, 7, 1]
    s = G.Stream()
    rope = G.Rope(hd, 1e4)
    ws = G.Buffer(max(16, G.paged_attn_workspace_bytes(c.kv, c.batch, n_head)))
    cache = [[np.zeros((0, n_kv, hd)), np.zeros((0, n_kv, hd))] for _ in lens]

    def layer(batch, n, x, qkv, out):
        G.matmul(W, qkv, nb=n, x=x, path=1, stream=s.ptr)
        p = qkv.ptr
        G.paged_append(c.kv, batch, p + 4 * n_head * hd, p + 4 * (n_head + n_kv) * hd, q=p, q_out=p, n_head=n_head, rope=rope, q_stride=total,
                       q_out_stride=total, k_stride=total, v_stride=total, stream=s.ptr)
        G.paged_attn(c.kv, batch, p, n_head, out, scale=0.2, softcap=30.0, ws=ws, q_stride=total, stream=s.ptr)

    def check(batch, new, qkv, out):
        n = sum(new)
        rows = qkv.download(np.float32, (n, total))
        q = rows[:, :n_head * hd].reshape(n, n_head, hd)
        got = out.download(np.float32, (n, n_head, hd))
        k, v = G.Buffer(n * n_kv * hd * 4), G.Buffer(n * n_kv * hd * 4)
        G.paged_read(c.kv, batch, k, v)
        k, v = (b.download(np.float32, (n, n_kv, hd)).astype(np.float64) for b in (k, v))
        raw_k = rows[:, n_head * hd:(n_head + n_kv) * hd].reshape(n, n_kv, hd)
        t0 = 0
        for i, m in enumerate(new):
            cache[i][0] = np.concatenate([cache[i][0], k[t0:t0 + m]])
            cache[i][1] = np.concatenate([cache[i][1], v[t0:t0 + m]])
            size = len(cache[i][0])
            at = n_pre + np.arange(size - m, size)
            turned = U.turn(raw_k[t0:t0 + m], at, hd, 1e4)
            step = np.abs(turned).max() / {F16: 1024, Q8_0: 127, Q4_0: 7}[t]
            assert np.abs(turned - k[t0:t0 + m]).max() <= step
            for j in range(m):
                for h in range(n_head):
                    kk, vv = (np.concatenate([c.shared[w][:, h // 2], cache[i][w][:, h // 2]]) for w in (0, 1))
                    want, tol = U.attend(q[t0 + j, h], kk, vv, n_pre + size - m + j, 0.2, 30.0)
                    assert np.all(np.abs(got[t0 + j, h] - want) <= tol)
            t0 += m
        assert c.kv.status() == 0

    n = sum(lens)
    x = G.Buffer.from_array(c.rng.standard_normal((n, width)).astype(np.float32))
    qkv, out = G.Buffer(n * total * 4), G.Buffer(n * n_head * hd * 4)
    c.d["lens"].upload(np.asarray(lens + [0], np.int32))
    layer(c.batch, n, x, qkv, out)
    s.synchronize()
    check(c.batch, lens, qkv, out)
    batch = G.PagedBatch(3, 3, c.d["lens"], c.d["table"], c.stride, 40, n_prefix=n_pre, prefix=c.d["pre"])
    ws = G.Buffer(max(16, G.paged_attn_workspace_bytes(c.kv, batch, n_head)))
    x1, qkv1, out1 = G.Buffer(3 * width * 4), G.Buffer(3 * total * 4), G.Buffer(3 * n_head * hd * 4)
    x1.upload(np.zeros((3, width), np.float32))
    G.matmul(W, qkv1, nb=3, x=x1, path=1, stream=s.ptr)              # its scratch, before the capture
    s.synchronize()
    g = G.Graph(s.ptr, lambda: layer(batch, 3, x1, qkv1, out1))
    for step in range(5):
        lens = [n + 1 for n in lens]
        c.d["lens"].upload(np.asarray(lens + [0], np.int32))
        x1.upload(c.rng.standard_normal((3, width)).astype(np.float32))
        g.launch(s.ptr)
        s.synchronize()
        check(batch, [1, 1, 1], qkv1, out1)
