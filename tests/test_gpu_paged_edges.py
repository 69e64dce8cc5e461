"""The paged KV cache's calls at the edges of what the header allows: offsets that
are not a whole batch's, and offsets that are wrong."""
import numpy as np
import pytest

from paged_util import F16, Q4_0, Q8_0, Case, turn, values

pytestmark = pytest.mark.gpu
TYPES = [F16, Q8_0, Q4_0]
IDS = ["f16", "q8_0", "q4_0"]


def _guarded(G, c, scale, **more):
    """Attention into rows with more behind them, which have to stay."""
    out = G.Buffer.from_array(np.full((c.n_tok + 5, c.n_head, c.hd), 7.5, np.float32))
    need = G.paged_attn_workspace_bytes(c.kv, c.batch, c.n_head)
    ws = G.Buffer.from_array(np.full(need + 4096, 0x7f, np.uint8))
    G.paged_attn(c.kv, c.batch, c.d["q"], c.n_head, out, scale=scale, ws=ws.ptr, **more)
    got = out.download(np.float32, (c.n_tok + 5, c.n_head, c.hd))
    assert np.all(got[c.n_tok:] == 7.5) and np.all(ws.download(np.uint8, (ws.nbytes,))[need:] == 0x7f)
    return got[:c.n_tok]


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("n_prefix", [0, 40, 700])
@pytest.mark.parametrize("heads", [(2, 1), (40, 2)])
@pytest.mark.parametrize("offs,good", [
    ([0, 2, 9, 6, 8], 2),                                  # past n_tok, then descending
    ([0, 5, 2, 6, 3], 5),                                  # tokens of two sequences each
    ([0, 8, 0, 8, 0], 8),
    ([-1, 2, 3, 4, 8], 0),
    ([1 << 30, 2, 3, 4, 8], 0),
    ([0, 1, 2, 5, -1 << 31], 5),
])
def test_rows_from_torn_offsets_on_read_as_nan(gpu, t, n_prefix, heads, offs, good):
    new = [offs[i + 1] - offs[i] if 0 <= offs[i] <= offs[i + 1] <= 8 else 1 for i in range(4)]
    c = Case(gpu, t, *heads, 64, 16, [300, 290, 310, 200], new=new, pad=8 - sum(new) if sum(new) < 8 else 0, n_prefix=n_prefix, seed=60)
    c.n_tok = c.batch.struct.n_tok = 8
    c.q = c.rng.standard_normal((8, heads[0], 64)).astype(np.float32)
    c.d["q"] = gpu.Buffer.from_array(c.q)
    c.off = np.asarray(offs, np.int32)
    c.d["off"].upload(c.off)
    last = next(s for s in range(4) if not 0 <= offs[s] <= offs[s + 1] <= 8)
    c.new, c.lens = new[:last], c.lens[:last]
    want, tol = c.expect(0.125)
    got = _guarded(gpu, c, 0.125)
    assert c.kv.status() == gpu.PAGED_BAD_BATCH
    assert np.all(np.abs(got[:good] - want[:good]) <= tol[:good])
    assert np.isnan(got[good:]).all()


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("n_prefix,window", [(0, 0), (40, 0), (700, 100)])
def test_offsets_torn_behind_many_sequences(gpu, t, n_prefix, window):
    # the first bad offset lies past the 64 sequences that are looked at at once
    n = 150
    new = [i % 3 for i in range(n)]
    c = Case(gpu, t, 4, 2, 64, 16, [v + 7 * i % 90 for i, v in enumerate(new)], new=new, n_prefix=n_prefix, seed=61)
    want, tol = c.expect(0.125, window=window)
    off = c.off.copy()
    off[132] = off[130] - 1
    c.d["off"].upload(off)
    got, end = _guarded(gpu, c, 0.125, window=window), int(off[131])
    assert c.kv.status() == gpu.PAGED_BAD_BATCH
    assert np.all(np.abs(got[:end] - want[:end]) <= tol[:end]) and np.isnan(got[end:]).all()


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("n_prefix", [0, 40])
@pytest.mark.parametrize("lens,new", [([300, 290, 310, 200], [4, 1, 2, 1]), ([90, 150, 60, 70], [60, 70, 30, 2])])
def test_a_part_of_a_batch(gpu, t, n_prefix, lens, new):
    # sequences 1 and 2 of four, over the same arrays: rows of the others are left
    c = Case(gpu, t, 4, 2, 64, 16, lens, new=new, pad=1, n_prefix=n_prefix, seed=62)
    want, tol = c.expect(0.125)
    s = c.batch.struct
    s.n_seq, s.q_off_dev, s.len_dev, s.table_dev = 2, s.q_off_dev + 4, s.len_dev + 4, s.table_dev + 4 * c.stride
    got = _guarded(gpu, c, 0.125)
    a, b = int(c.off[1]), int(c.off[3])
    assert np.all(np.abs(got[a:b] - want[a:b]) <= tol[a:b])
    assert np.all(got[:a] == 7.5) and np.all(got[b:] == 7.5)
    assert c.kv.status() == 0


# -------------------------------------------------------------- pages given away
@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("hd,n_head,n_kv", [(64, 4, 2), (128, 8, 4), (256, 4, 2), (512, 2, 1), (64, 40, 2)])
@pytest.mark.parametrize("page", [16, 48])
@pytest.mark.parametrize("new", [None, [2, 1, 3, 1], [70, 100, 1, 64]])
def test_pages_before_the_window_may_be_given_away(gpu, t, hd, n_head, n_kv, page, new):
    window, lens = 50, [150, 113, 99, 49]
    c = Case(gpu, t, n_head, n_kv, hd, page, lens, new=[min(n, m) for n, m in zip(new, lens)] if new else None, seed=hd + page)
    gone = 0
    for s, (n, m) in enumerate(zip(c.lens, c.new)):
        k = max(0, n - m + 1 - window) // page             # whole pages that no token of the call attends
        c.table[s, :k] = -1 if s % 2 else c.pool.n_pages
        gone += k
    assert gone
    c.d["table"].upload(c.table)
    c.check(window=window)
    c.check(window=window, cap=20.0)


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("n_seq", [1, 30])
@pytest.mark.parametrize("own", [60, 200])
def test_a_prefix_before_all_windows_may_be_given_away(gpu, t, n_seq, own):
    # its last pages are still attended by the shorter sequences
    c = Case(gpu, t, 4, 2, 64, 16, [own + i % 7 for i in range(n_seq)], n_prefix=150, seed=63)
    k = max(0, 150 + own - 100) // 16
    c.prefix[:k] = -1
    c.d["pre"].upload(c.prefix)
    c.check(window=100)


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("hd,n_head,n_kv", [(64, 4, 2), (256, 4, 2), (512, 2, 1)])
@pytest.mark.parametrize("n,window", [(3, 0), (90, 0), (90, 20), (6, 20)])
def test_a_bad_page_reaches_only_the_rows_that_attend_it(gpu, t, hd, n_head, n_kv, n, window):
    # a chunk of n tokens; the page of positions 112 .. 127 is wrong
    c = Case(gpu, t, n_head, n_kv, hd, 16, [130, 130], new=[n, n], seed=64)
    c.table[0, 7] = -5
    c.d["table"].upload(c.table)
    want, tol = c.expect(0.1, window=window)
    got = c.attn(0.1, window=window)
    hit = np.zeros(c.n_tok, bool)
    pos = 130 - n + np.arange(n)
    hit[:n] = (pos >= 112) & ((pos - window < 127) if window else True)
    assert np.isnan(got[hit]).all()
    assert np.all(np.abs(got - want)[~hit] <= tol[~hit])
    assert c.kv.status() == gpu.PAGED_BAD_PAGE


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("n_prefix", [0, 40])
@pytest.mark.parametrize("heads", [(2, 1), (40, 2)])
def test_the_largest_window_with_padded_slots(gpu, t, n_prefix, heads):
    # tokens before position 0 among others, and a window as large as an int
    for lens, new in (([0, 5, 40], [3, 9, 40]), ([5, 70, 0], [9, 60, 2]), ([0, 3, 2, 60], [2, 4, 5, 1])):
        c = Case(gpu, t, *heads, 64, 16, lens, new=new, n_prefix=n_prefix, seed=65)
        for window in ((1 << 31) - 1, (1 << 31) - 3, n_prefix + max(lens), n_prefix + max(lens) - 1):
            c.check(window=window)


# ------------------------------------------------------------ fused rows
@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("new", [None, [30, 2, 60]])
def test_outputs_beside_the_queries_of_a_fused_row(gpu, t, new):
    G = gpu
    c = Case(G, t, 4, 2, 64, 16, [70, 5, 90], new=new, pad=1 if new else 0, n_prefix=20, seed=66)
    w = 2 * 256 + 12
    x = np.full((c.n_tok, w), 3.0, np.float32)
    x[:, :256] = c.q.reshape(c.n_tok, 256)
    b = G.Buffer.from_array(x)
    G.paged_attn(c.kv, c.batch, b, 4, b.ptr + 4 * 260, scale=0.125, q_stride=w, out_stride=w)
    got = b.download(np.float32, x.shape)
    want, tol = c.expect(0.125)
    n = c.n_tok - c.pad
    assert np.all(np.abs(got[:n, 260:516].reshape(n, 4, 64) - want[:n]) <= tol[:n])
    got[:n, 260:516] = 3.0
    assert np.array_equal(got, x)


@pytest.mark.parametrize("n_seq,n_tok", [(0, 0), (3, 0), (0, 3)])
def test_an_empty_batch_does_nothing(gpu, n_seq, n_tok):
    G = gpu
    kv = G.PagedKV(Q8_0, 2, 64, 16, 4)
    for n_prefix in (0, 20):
        b = G.PagedBatch(n_seq, n_tok, None, None, 2, 32, n_prefix=n_prefix)
        for n_head in (2, 40):
            G.paged_append(kv, b, None, None, n_head=n_head, rope=G.Rope(64, 1e4))
            G.paged_attn(kv, b, None, n_head, None)
            G.paged_read(kv, b)
    out = G.Buffer.from_array(np.full((3, 2, 64), 7.5, np.float32))
    G.paged_attn(kv, b, out.ptr, 2, out.ptr)
    assert np.all(out.download(np.float32, (3, 2, 64)) == 7.5) and kv.status() == 0


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("new", [[4, 1, 2, 1], [300, 700, 600, 500]])
def test_append_and_read_of_a_part_of_a_batch(gpu, t, new):
    # rows of sequences 1 and 2 of four are stored, rotated and read, the others left, and nothing is flagged
    G = gpu
    c = Case(G, t, 2, 1, 64, 16, [n + 20 for n in new], new=new, pad=2, seed=67)
    s = c.batch.struct
    s.n_seq, s.q_off_dev, s.len_dev, s.table_dev = 2, s.q_off_dev + 4, s.len_dev + 4, s.table_dev + 4 * c.stride
    a, b = int(c.off[1]), int(c.off[3])
    k, v = (c.rng.standard_normal((c.n_tok, 1, 64)).astype(np.float32) for _ in range(2))
    kb, vb, qo = G.Buffer.from_array(k), G.Buffer.from_array(v), G.Buffer.from_array(np.full_like(c.q, 7.5))
    G.paged_append(c.kv, c.batch, kb, vb, q=c.d["q"], q_out=qo, n_head=2, rope=G.Rope(64, 1e4))
    ko, vo = (G.Buffer.from_array(np.full(k.shape, 7.5, np.float32)) for _ in range(2))
    G.paged_read(c.kv, c.batch, ko, vo)
    assert c.kv.status() == 0
    pos = np.zeros(c.n_tok)
    pos[a:b] = np.concatenate([c.lens[i] - c.new[i] + np.arange(c.new[i]) for i in (1, 2)])
    q, gk, gv = qo.download(np.float32, c.q.shape), ko.download(np.float32, k.shape), vo.download(np.float32, v.shape)
    for x in (q, gk, gv):
        assert np.all(x[:a] == 7.5) and np.all(x[b:] == 7.5)
    want = turn(c.q, pos, 64, 1e4)
    assert np.all(np.abs(q - want)[a:b] <= np.abs(c.q).max() * 2.0 ** -20)
    assert np.array_equal(gv[a:b], values(t, v)[a:b].astype(np.float32))
    changed = (c.kv.v.download(np.uint8, c.pool.v.shape) != c.pool.v).any(1)
    assert set(np.flatnonzero(changed)) <= {int(p) for i in (1, 2) for p in c.table[i]}


@pytest.mark.parametrize("t", TYPES, ids=IDS)
def test_no_status_word(gpu, t):
    # a cache without one: bad pages and offsets are read as they are with it
    c = Case(gpu, t, 4, 2, 64, 16, [60, 40, 20], new=[1, 2, 1], n_prefix=20, seed=68)
    c.table[0, 1] = -1
    c.d["table"].upload(c.table)
    c.kv.struct.status_dev = None
    want, tol = c.expect(0.1)
    got = c.attn(0.1)
    assert np.isnan(got[0]).all() and np.all(np.abs(got[1:] - want[1:]) <= tol[1:])
    c.d["off"].upload(np.asarray([0, 1, 9, 4], np.int32))
    got = c.attn(0.1)
    assert np.isnan(got).all()
    k = gpu.Buffer.from_array(c.rng.standard_normal((4, 2, 64)).astype(np.float32))
    gpu.paged_append(c.kv, c.batch, k, k)
    gpu.synchronize()


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
def test_append_rounds_as_kv_store(gpu, t, hd):
    # every bit that a stored row's values depend on, of blocks of any size
    G, n = gpu, 96
    c = Case(G, t, 1, 1, hd, 16, [n], new=[n], seed=69)
    x = (c.rng.standard_normal((n, 1, hd)) * np.exp2(c.rng.integers(-40, 20, (n, 1, hd // 32))).repeat(32, -1)).astype(np.float32)
    x[1] = 0
    x[2] = np.float32(1e-42)
    x[3] *= np.float32(1e30)
    x[4] = np.sign(x[4])
    x[5, 0, :32] = np.arange(-16, 16) / 16
    x[6] = -np.abs(x[6])
    x[7, 0, ::2] = -x[7, 0, 1::2]
    b = G.Buffer.from_array(x)
    G.paged_append(c.kv, c.batch, b, b)
    size = {F16: 2 * hd, Q8_0: hd // 32 * 34, Q4_0: hd // 32 * 18}[t]
    flat = G.Buffer(n * size)
    G.kv_store(t, b, flat, hd, n)
    G.synchronize()
    want = flat.download(np.uint8, (n, size))
    c.pool.k, c.pool.v = c.kv.k.download(np.uint8, c.pool.k.shape), c.kv.v.download(np.uint8, c.pool.v.shape)
    row = hd * 2 if t == F16 else hd if t == Q8_0 else hd // 2
    for p in range(n):
        pg, slot = c.table[0, p // 16], p % 16
        for raw, at in ((c.pool.k, "k"), (c.pool.v, "v")):
            bytes_ = raw[pg, slot * row:(slot + 1) * row]
            if t == F16:
                assert np.array_equal(bytes_, want[p])
                continue
            scales = raw[pg, 16 * row + slot * (hd // 16):16 * row + (slot + 1) * (hd // 16)].reshape(-1, 2)
            blocks = want[p].reshape(hd // 32, -1)
            assert np.array_equal(scales, blocks[:, :2]), (p, at)
            if t == Q8_0:
                q = bytes_[getattr(c.pool, at + "8")].astype(np.int32) - 128
                w = blocks[:, 2:].view(np.int8).astype(np.int32).reshape(-1)
            else:
                q = np.stack([bytes_ & 15, bytes_ >> 4], -1).reshape(-1)[getattr(c.pool, at + "4")].astype(np.int32)
                w = np.concatenate([blocks[:, 2:] & 15, blocks[:, 2:] >> 4], 1).astype(np.int32).reshape(-1)
            # of a zero scale (one below 2^-25) every quant is the value 0: 1 / d may be infinite there
            held = np.repeat(scales.copy().view(np.float16)[:, 0] != 0, 32)
            assert np.array_equal(q[held], w[held]), (p, at)
