"""Drafts that are trees over the paged KV cache, against a plain model in float64
(tests/tree_util.py): attention under masks, masks and depths from parents, rotation
by depth, the accepted path, and its rows moved together."""
import numpy as np
import pytest

from paged_util import F16, Q4_0, Q8_0, Pool, turn, values
from tree_util import TreeCase, ancestry, pack, random_parents, walk

pytestmark = pytest.mark.gpu
TYPES = [F16, Q8_0, Q4_0]


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd,n_head,n_kv", [(64, 4, 2), (128, 8, 2), (256, 4, 2), (512, 2, 1)])
@pytest.mark.parametrize("new", [[1], [2, 1], [5, 3], [8, 16], [17, 4], [33, 31, 1], [64]])
def test_trees(gpu, t, hd, n_head, n_kv, new):
    TreeCase(gpu, t, n_head, n_kv, hd, 16, [n + 13 + 9 * i for i, n in enumerate(new)], new, seed=hd + len(new)).check()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
def test_trees_of_one_query_head(gpu, t, hd):
    TreeCase(gpu, t, 1, 1, hd, 32, [70, 40], [11, 20], seed=3).check()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("first", [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100])
def test_where_the_new_tokens_begin(gpu, t, first):
    TreeCase(gpu, t, 4, 2, 64, 16, [first + 7, first + 40], [7, 40], seed=first).check()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,words", [(31, 1), (32, 1), (33, 2), (96, 3), (97, 4), (200, 7)])
def test_words(gpu, t, n, words):
    TreeCase(gpu, t, 2, 2, 64, 16, [n + 21], [n], words=words, seed=n).check()


def test_the_most_words(gpu):
    TreeCase(gpu, F16, 1, 1, 64, 64, [1024 + 5], [1024], words=32, seed=1).check()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("new", [[6, 1], [40, 3]])
@pytest.mark.parametrize("first", [0, 20])
def test_masks_of_any_kind(gpu, t, new, first):
    # later tokens, not the own one, none at all, tokens that the sequence does not have
    rng = np.random.default_rng(5)
    sets = []
    for n in new:
        for i in range(n):
            sets.append([set(), set(range(n)), {j for j in range(64) if rng.random() < 0.4}, {n - 1}, {0}, {63}][(i + first) % 6])
    TreeCase(gpu, t, 4, 2, 64, 16, [n + first for n in new], new, words=2, sets=sets, seed=2).check()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("new", [[6], [24, 9]])
@pytest.mark.parametrize("n_prefix", [0, 37])
@pytest.mark.parametrize("window", [1, 2, 16, 33, 64, 1000])
def test_window(gpu, t, new, n_prefix, window):
    TreeCase(gpu, t, 4, 2, 64, 16, [n + 50 for n in new], new, n_prefix=n_prefix, seed=window).check(window=window)


@pytest.mark.parametrize("new", [[4, 7], [30, 2]])
@pytest.mark.parametrize("window", [0, 5, 40])
def test_depths_of_any_size_count_as_the_nearest(gpu, new, window):
    n = sum(new)
    depths = [[-5, 10 ** 6, 2 ** 31 - 1, -2 ** 31, 1][i % 5] for i in range(n)]
    TreeCase(gpu, F16, 2, 1, 64, 16, [n + 30 for n in new], new, depths=depths, n_prefix=20, seed=4).check(window=window)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("cap", [0.5, 30.0])
@pytest.mark.parametrize("new", [[7, 2], [40]])
def test_cap(gpu, t, cap, new):
    TreeCase(gpu, t, 8, 2, 128, 32, [n + 60 for n in new], new, seed=6).check(cap=cap)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd,n_head,n_kv,new", [(64, 4, 2, [3, 1, 5]), (128, 8, 2, [20, 5]), (256, 8, 4, [40, 9]), (512, 4, 2, [3, 2])])
@pytest.mark.parametrize("n_prefix", [1, 40, 300])
def test_prefix(gpu, t, hd, n_head, n_kv, new, n_prefix):
    TreeCase(gpu, t, n_head, n_kv, hd, 16, [n + 6 for n in new], new, n_prefix=n_prefix, seed=7).check()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("new", [[5], [23], [70]])
def test_long(gpu, t, new):
    TreeCase(gpu, t, 4, 1, 128, 64, [n + 2500 for n in new], new, seed=8).check()


@pytest.mark.parametrize("new", [[6] * 40, [20] * 24, [3] * 300])
def test_many_sequences(gpu, new):
    TreeCase(gpu, F16, 2, 1, 64, 16, [n + (7 * i) % 90 for i, n in enumerate(new)], new, seed=9).check()


@pytest.mark.parametrize("t", TYPES)
def test_padded_slots_and_rows_behind(gpu, t):
    # sequences without positions, and tokens before position 0 (no room for all of a draft)
    c = TreeCase(gpu, t, 4, 2, 64, 16, [0, 40, 3, 0], [1, 9, 7, 5], pad=3, seed=10)
    c.check()
    c = TreeCase(gpu, t, 4, 2, 64, 16, [30, 12], [24, 40], pad=2, seed=11)
    c.check()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("new", [[6, 4], [40]])
def test_chains_attend_as_rows_of_tokens(gpu, t, new):
    c = TreeCase(gpu, t, 4, 2, 128, 16, [n + 77 for n in new], new, sets=[set(range(i + 1)) for n in new for i in range(n)],
                 depths=[i for n in new for i in range(n)], seed=12)
    want, tol = super(TreeCase, c).expect(128 ** -0.5)
    got = c.attn(128 ** -0.5)
    assert (np.abs(got - want) <= tol).all()
    same = c.G.Buffer(got.nbytes)
    c.G.paged_attn(c.kv, c.batch, c.d["q"], c.n_head, same, scale=128 ** -0.5)
    assert (np.abs(got - same.download(np.float32, got.shape)) <= 2 * tol).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("new", [[8], [44]])
@pytest.mark.parametrize("n_prefix", [0, 20])
def test_slots_that_a_row_does_not_attend_may_hold_anything(gpu, t, new, n_prefix):
    # new token 2 holds infinities: those that attend it get no finite value, the others their own
    c = TreeCase(gpu, t, 4, 2, 64, 16, [n + 20 for n in new], new, n_prefix=n_prefix, seed=13)
    clean = c.attn(0.125)
    slot = c.lens[0] - new[0] + 2
    page = c.table[0, slot // 16]
    for raw, n in ((c.pool.k, 128 if t == F16 else 4), (c.pool.v, 128 if t == F16 else 4)):
        for h in range(2):
            row = h * 16 + slot % 16
            at = row * 128 if t == F16 else 2 * 16 * (64 if t == Q8_0 else 32) + row * 4
            raw[page, at:at + n] = np.full(n // 2, 0x7c00, np.uint16).view(np.uint8)
    c._upload()
    c.tree = c.G.PagedTree(c.words, c.d.setdefault("mask", c.G.Buffer.from_array(pack(c.sets, c.words))),
                           c.d.setdefault("depth", c.G.Buffer.from_array(np.asarray(c.depths, np.int32))))
    got = c.attn(0.125)
    reads = np.array([2 in s for s in c.sets])
    assert not np.isfinite(got[reads]).all(-1).any()
    assert np.array_equal(got[~reads], clean[~reads])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("new", [[8, 3], [44, 20]])
def test_a_bad_page_reaches_only_the_rows_that_attend_it(gpu, t, new):
    c = TreeCase(gpu, t, 4, 2, 64, 16, [16 + n for n in new], new, seed=14)
    clean = c.attn(0.125)
    table = c.table.copy()
    table[0, -(-c.lens[0] // 16) - 1] = 10 ** 6               # the page of the last new tokens
    c.d["table"].upload(table)
    got = c.attn(0.125)
    lost = set(range((c.lens[0] - 1) // 16 * 16 - 16, new[0]))
    for i in range(new[0]):
        assert np.isnan(got[i]).all() if c.sets[i] & lost else np.array_equal(got[i], clean[i]), i
    assert np.array_equal(got[new[0]:], clean[new[0]:])
    assert c.kv.status() == gpu.PAGED_BAD_PAGE


def test_bad_lengths_and_offsets_are_flagged(gpu):
    c = TreeCase(gpu, F16, 4, 2, 64, 16, [30, 20, 25], [9, 5, 20], seed=15)
    want, tol = c.expect(0.125)
    near = lambda x, at: (np.abs(x[at] - want[at]) <= tol[at]).all()  # noqa: E731
    c.d["lens"].upload(np.array([30, 1000, 25, 0], np.int32))
    got = c.attn(0.125)
    assert np.isnan(got[9:14]).all() and near(got, slice(0, 9)) and near(got, slice(14, 34))
    assert c.kv.status() == gpu.PAGED_BAD_BATCH
    c.d["lens"].upload(np.array([30, 20, 25, 0], np.int32))
    c.d["off"].upload(np.array([0, 9, 7, 34], np.int32))
    got = c.attn(0.125)
    assert near(got, slice(0, 9)) and np.isnan(got[9:]).all()
    assert c.kv.status() == gpu.PAGED_BAD_BATCH


@pytest.mark.parametrize("new", [[5, 2], [50]])
def test_strides(gpu, new):
    G = gpu
    c = TreeCase(G, F16, 4, 2, 64, 16, [n + 33 for n in new], new, seed=16)
    want, row, w = c.attn(0.125), 4 * 64, 2 * 4 * 64 + 3
    both = np.full((c.n_tok, w), 5.0, np.float32)
    both[:, :row] = c.q.reshape(c.n_tok, row)
    at = G.Buffer.from_array(both)
    G.paged_attn_tree(c.kv, c.batch, c.tree, at, 4, at.ptr + 4 * (row + 1), scale=0.125, q_stride=w, out_stride=w)
    got = at.download(np.float32, both.shape)
    assert np.array_equal(got[:, row + 1:2 * row + 1].reshape(want.shape), want)
    keep = np.ones(w, bool)
    keep[row + 1:2 * row + 1] = False
    assert np.array_equal(got[:, keep], both[:, keep])


@pytest.mark.parametrize("new", [[5, 9], [50, 7]])
def test_runs_repeat_bit_for_bit(gpu, new):
    c = TreeCase(gpu, Q8_0, 8, 2, 128, 16, [n + 700 for n in new], new, n_prefix=90, seed=17)
    first = c.attn(0.1)
    assert all(np.array_equal(c.attn(0.1), first) for _ in range(3))


@pytest.mark.parametrize("new", [[7, 3], [60, 20]])
def test_graph_replays_with_other_trees(gpu, new):
    G = gpu
    c = TreeCase(G, F16, 4, 2, 64, 16, [n + 400 for n in new], new, seed=18)
    ws = G.Buffer(max(16, G.paged_attn_tree_workspace_bytes(c.kv, c.batch, 4)))
    out = G.Buffer(c.n_tok * 4 * 64 * 4)
    s = G.Stream()
    G.paged_attn_tree(c.kv, c.batch, c.tree, c.d["q"], 4, out, scale=0.125, ws=ws, stream=s.ptr)
    g = G.Graph(s.ptr, lambda: G.paged_attn_tree(c.kv, c.batch, c.tree, c.d["q"], 4, out, scale=0.125, ws=ws, stream=s.ptr))
    rng, full = np.random.default_rng(19), [x[:] for x in c.rows]
    for cut in (0, 100, 333, 5):
        c.lens = [n + 400 - cut for n in new]
        c.rows = [[w[:n] for w in x] for x, n in zip(full, c.lens)]
        parents = [random_parents(rng, n) for n in new]
        c.sets, c.depths = ([x for p in parents for x in ancestry(p)[i]] for i in (0, 1))
        c.d["lens"].upload(np.array(c.lens + [0], np.int32), s.ptr)
        c.d["mask"].upload(pack(c.sets, c.words), s.ptr)
        c.d["depth"].upload(np.array(c.depths, np.int32), s.ptr)
        g.launch(s.ptr)
        s.synchronize()
        got = out.download(np.float32, (c.n_tok, 4, 64))
        assert np.array_equal(got, c.attn(0.125)), cut
        c.check()


def test_calls_on_other_streams(gpu):
    G = gpu
    cases = [TreeCase(G, t, 4, 2, 128, 16, [300, 64], [20, 5], seed=30 + t) for t in TYPES]
    streams = [G.Stream() for _ in cases]
    ws = [G.Buffer(max(16, G.paged_attn_tree_workspace_bytes(c.kv, c.batch, 4))) for c in cases]
    outs = [G.Buffer(c.n_tok * 4 * 128 * 4) for c in cases]
    for _ in range(5):
        for c, s, w, o in zip(cases, streams, ws, outs):
            G.paged_attn_tree(c.kv, c.batch, c.tree, c.d["q"], 4, o, scale=0.1, ws=w, stream=s.ptr)
    for c, s, o in zip(cases, streams, outs):
        s.synchronize()
        want, tol = c.expect(0.1)
        assert np.all(np.abs(o.download(np.float32, want.shape) - want) <= tol)


# ------------------------------------------------------- masks, depths, append
def _batch(G, new, n_tok=None, lens=None, offs=None):
    off = np.concatenate([[0], np.cumsum(new)]).astype(np.int32) if offs is None else np.asarray(offs, np.int32)
    B = G.Buffer.from_array
    lens = B(np.asarray((lens if lens is not None else new) or [0], np.int32))
    table = B(np.zeros((max(1, len(new)), 1), np.int32))
    return G.PagedBatch(len(new), int(off[-1]) if n_tok is None else n_tok, lens, table, 1, 1 << 20, q_off=B(off))


def _build(G, new, parents, words, n_tok=None, offs=None):
    batch = _batch(G, new, n_tok, offs=offs)
    n = batch.struct.n_tok
    mask, depth = G.Buffer.from_array(np.full((n, words), 0xabcdef01, np.uint32)), G.Buffer.from_array(np.full(n, -9, np.int32))
    status = G.Buffer.from_array(np.zeros(1, np.int32))
    p = G.Buffer.from_array(np.asarray(parents + [-1] * (n - len(parents)), np.int32))
    G.paged_tree_build(batch, p, words, mask, depth, status)
    return mask.download(np.uint32, (n, words)), depth.download(np.int32, (n,)), int(status.download(np.int32, (1,))[0])


@pytest.mark.parametrize("new,words", [([1], 1), ([32], 1), ([33, 1, 0, 5], 2), ([64] * 9, 2), ([3] * 500, 1), ([1024, 7], 32), ([200], 32)])
def test_build(gpu, new, words):
    rng = np.random.default_rng(words)
    trees = [random_parents(rng, n) for n in new]
    mask, depth, flags = _build(gpu, new, sum(trees, []), words, n_tok=sum(new) + 2)
    n = sum(new)
    assert np.array_equal(mask[:n], np.concatenate([pack(ancestry(p)[0], words) for p in trees]))
    assert depth[:n].tolist() == sum((ancestry(p)[1] for p in trees), [])
    assert (mask[n:] == 0xabcdef01).all() and (depth[n:] == -9).all() and flags == 0


def test_build_of_a_chain(gpu):
    mask, depth, flags = _build(gpu, [1024], list(range(-1, 1023)), 32)
    assert np.array_equal(mask, pack([set(range(i + 1)) for i in range(1024)], 32)) and depth.tolist() == list(range(1024)) and flags == 0


@pytest.mark.parametrize("bad", [3, 4, 100, -2, -2 ** 31, 2 ** 31 - 1])
def test_a_bad_parent_counts_as_none(gpu, bad):
    parents, plain = [-1, 0, 1, bad, 3, 2], [-1, 0, 1, -1, 3, 2]
    mask, depth, flags = _build(gpu, [6, 2], parents + [-1, 0], 1)
    sets, depths = ancestry(plain)
    assert np.array_equal(mask, np.concatenate([pack(sets, 1), [[1], [3]]])) and depth.tolist() == depths + [0, 1]
    assert flags == gpu.PAGED_BAD_BATCH


def test_more_tokens_than_bits(gpu):
    mask, depth, flags = _build(gpu, [70, 2], list(range(-1, 69)) + [-1, 0], 2)
    assert np.array_equal(mask[:64], pack([set(range(i + 1)) for i in range(64)], 2)) and depth[:64].tolist() == list(range(64))
    assert not mask[64:70].any() and not depth[64:70].any() and mask[70:].tolist() == [[1, 0], [3, 0]] and flags == gpu.PAGED_BAD_BATCH


def test_build_one_token_each(gpu):
    G = gpu
    B = G.Buffer.from_array
    batch = G.PagedBatch(5, 5, None, None, 0, 0)
    mask, depth, status = B(np.zeros(5, np.uint32)), B(np.full(5, 9, np.int32)), B(np.zeros(1, np.int32))
    G.paged_tree_build(batch, B(np.full(5, -1, np.int32)), 1, mask, depth, status)
    assert mask.download(np.uint32, (5,)).tolist() == [1] * 5 and depth.download(np.int32, (5,)).tolist() == [0] * 5
    assert status.download(np.int32, (1,))[0] == 0


def test_build_flags_torn_offsets(gpu):
    assert _build(gpu, [3, 2], [-1] * 5, 1, n_tok=5, offs=[0, 4, 2])[2] == gpu.PAGED_BAD_BATCH
    assert _build(gpu, [3, 2], [-1] * 5, 1, n_tok=5, offs=[0, 3, 9])[2] == gpu.PAGED_BAD_BATCH
    assert _build(gpu, [3, 2], [-1] * 5, 1, n_tok=5, offs=[-1, 3, 5])[2] == gpu.PAGED_BAD_BATCH


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n_prefix", [0, 1000])
def test_append_turns_by_depth(gpu, t, n_prefix):
    G, hd, n_head, n_kv = gpu, 64, 4, 2
    c = TreeCase(G, t, n_head, n_kv, hd, 16, [30, 8, 4], [9, 8, 6], seed=20)
    rng = np.random.default_rng(21)
    k, v = (rng.standard_normal((23, n_kv, hd)).astype(np.float32) for _ in range(2))
    q_out, batch = G.Buffer.from_array(np.full((23, n_head, hd), 3.0, np.float32)), c.batch
    batch.struct.n_prefix = n_prefix
    G.paged_append_tree(c.kv, batch, G.PagedTree(c.words, None, c.d["depth"]), G.Buffer.from_array(k), G.Buffer.from_array(v), q=c.d["q"],
                        q_out=q_out, n_head=n_head, rope=G.Rope(hd, 1e4))
    pool = Pool(t, n_kv, hd, 16, c.pool.n_pages)
    pool.k, pool.v = (b.download(np.uint8, c.pool.k.shape) for b in (c.kv.k, c.kv.v))
    got = q_out.download(np.float32, (23, n_head, hd))
    for s, (n, size) in enumerate(zip(c.new, c.lens)):
        for i in range(n):
            tok, slot = c.off[s] + i, size - n + i
            if slot < 0:
                assert (got[tok] == 3.0).all()
                continue
            pos = n_prefix + size - n + c.depths[tok]
            # an fp32 turn: two products and a sum, of angles rounded to fp32
            assert np.abs(got[tok] - turn(c.q[tok:tok + 1], [pos], hd, 1e4)[0]).max() <= 8 * 2.0 ** -24 * np.abs(c.q[tok]).max()
            turned = turn(k[tok:tok + 1], [pos], hd, 1e4)[0]
            for h in range(n_kv):
                pg = c.table[s, slot // 16]
                # the cache's rounding of a block: half a step of its largest (f16 2^-11, q8_0 1 / 254, q4_0 1 / 8 where it is cut at 7)
                step = {F16: 2.0 ** -11, Q8_0: 1 / 254 + 2.0 ** -11, Q4_0: 1 / 8 + 2.0 ** -11}[t] + 2.0 ** -20
                for value, x in ((False, turned[h]), (True, v[tok, h])):
                    top = np.abs(x).reshape(-1, 32).max(1).repeat(32) if t != F16 else np.abs(x) + 2.0 ** -14
                    assert (np.abs(pool.get(value, pg, slot % 16, h) - x) <= step * top).all()
    assert c.kv.status() == 0


# ------------------------------------------------------------ accept and keep
def _accept(G, new, lens, parents, tokens, choice, most, offs=None, max_len=1 << 20, n_tok=None):
    B = G.Buffer.from_array
    batch = _batch(G, new, n_tok=n_tok, lens=lens, offs=offs)
    batch.struct.max_len = max_len
    s, arrays = len(new), [B(np.asarray(x or [0], np.int32)) for x in (parents, tokens, choice)]
    n_keep, keep, nxt, out = (B(np.full(m, 99, np.int32)) for m in (s, s * most, s, s))
    status = B(np.zeros(1, np.int32))
    G.paged_tree_accept(batch, *arrays, most, n_keep, keep, next_out=nxt, len_out=out, status=status)
    return (n_keep.download(np.int32, (s,)).tolist(), keep.download(np.int32, (s, most)).tolist(), nxt.download(np.int32, (s,)).tolist(),
            out.download(np.int32, (s,)).tolist(), int(status.download(np.int32, (1,))[0]))


@pytest.mark.parametrize("new,most", [([1], 1), ([8], 8), ([8, 1, 30, 0, 64], 5), ([200, 65], 40), ([12] * 300, 4), ([1024], 1024)])
@pytest.mark.parametrize("vocab", [1, 2, 4])
def test_accept(gpu, new, most, vocab):
    rng = np.random.default_rng(most + vocab)
    parents = [random_parents(rng, n) if vocab > 1 else list(range(-1, n - 1)) for n in new]
    tokens, choice = ([rng.integers(0, vocab, n).tolist() for n in new] for _ in range(2))
    lens = [n + 5 for n in new]
    want = [walk(*x, most) for x in zip(parents, tokens, choice)]
    got = _accept(gpu, new, lens, sum(parents, []), sum(tokens, []), sum(choice, []), most)
    assert got[0] == [len(p) for p, _ in want]
    assert got[1] == [p + [-1] * (most - len(p)) for p, _ in want]
    assert got[2] == [x for _, x in want] and got[3] == [5 + len(p) for p, _ in want] and got[4] == 0


def test_accept_of_sequences_without_room(gpu):
    n_keep, keep, nxt, out, flags = _accept(gpu, [3, 1, 2, 2], [2, 0, 2, 40], [-1, 0, 1, -1, -1, 0, -1, 0], [0] * 8, [0] * 8, 3, max_len=30)
    assert n_keep == [0, 0, 2, 0] and keep == [[-1] * 3, [-1] * 3, [0, 1, -1], [-1] * 3] and nxt == [-1, -1, 0, -1] and out == [0, 0, 2, 0]
    assert flags == gpu.PAGED_BAD_BATCH


def test_accept_of_torn_offsets(gpu):
    n_keep, _, nxt, out, flags = _accept(gpu, [2, 2, 1], [9, 9, 9], [-1, 0, -1, 0, -1], [0] * 5, [0] * 5, 2, offs=[0, 2, 1, 5], n_tok=5)
    assert n_keep[:2] == [2, 0] and nxt[1] == -1 and out[1] == 0 and flags == gpu.PAGED_BAD_BATCH


def _caches(G, t, n_kv, hd, page, n_pages, n, seed=0):
    rng = np.random.default_rng(seed)
    pools, kvs = [], []
    for _ in range(n):
        p = Pool(t, n_kv, hd, page, n_pages)
        p.k, p.v = (rng.integers(0, 256, p.k.shape, np.uint8) for _ in range(2))
        pools.append(p)
        kvs.append(G.PagedKV(t, n_kv, hd, page, n_pages, k=G.Buffer.from_array(p.k), v=G.Buffer.from_array(p.v)))
    return pools, kvs, G.PagedCaches(kvs)


def _rows(pool, raw):
    """Views [page, head, slot, bytes] of a pool's rows, and of their scales."""
    n = (2 if pool.t == F16 else 1 if pool.t == Q8_0 else 0.5) * pool.hd
    n = int(n)
    h, p = pool.n_kv, pool.page
    rows = raw[:, :h * p * n].reshape(-1, h, p, n)
    return [rows] if pool.t == F16 else [rows, raw[:, h * p * n:].reshape(-1, h, p, pool.hd // 16)]


def _moved(pool, table, first, keep):
    """The pool's bytes after a sequence's rows first + keep[k] went to first + k."""
    for raw in (pool.k, pool.v):
        for x in _rows(pool, raw):
            old = x.copy()
            for k, j in enumerate(keep):
                a, b = first + j, first + k
                x[table[b // pool.page], :, b % pool.page] = old[table[a // pool.page], :, a % pool.page]


def _same(pools, kvs):
    for p, kv in zip(pools, kvs):
        assert np.array_equal(kv.k.download(np.uint8, p.k.shape), p.k) and np.array_equal(kv.v.download(np.uint8, p.v.shape), p.v)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd,n_kv,page", [(64, 3, 16), (128, 8, 48), (256, 1, 32), (512, 2, 16)])
@pytest.mark.parametrize("n_cache", [1, 3])
def test_keep(gpu, t, hd, n_kv, page, n_cache):
    G = gpu
    new, lens = [9, 40, 1, 0, 16], [30, 40, 17, 5, 100]
    keeps = [[0, 3, 4, 8], [1, 5, 6, 7, 8, 9, 10, 20, 33, 38, 39], [0], [], list(range(16))]
    _keep_case(G, t, hd, n_kv, page, n_cache, new, lens, keeps)


def _keep_case(G, t, hd, n_kv, page, n_cache, new, lens, keeps, most=None, flags=0, given=None):
    most = most or max(len(k) for k in keeps) + 1
    need = [-(-n // page) for n in lens]
    ids = np.random.default_rng(1).permutation(sum(need) + 2)
    table = np.full((len(new), max(need)), -3, np.int32)
    for i, n in enumerate(need):
        table[i, :n] = ids[sum(need[:i]):sum(need[:i]) + n]
    pools, kvs, caches = _caches(G, t, n_kv, hd, page, len(ids), n_cache, seed=hd)
    B = G.Buffer.from_array
    off = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    batch = G.PagedBatch(len(new), int(off[-1]), B(np.asarray(lens, np.int32)), B(table), table.shape[1], max(lens), q_off=B(off))
    given = given or keeps
    n_keep, keep = B(np.asarray([len(k) for k in given], np.int32)), B(np.asarray([list(k) + [-1] * (most - len(k)) for k in given], np.int32))
    G.paged_keep(caches, batch, n_keep, keep, most)
    for p in pools:
        for s, k in enumerate(keeps):
            _moved(p, table[s], lens[s] - new[s], k)
    _same(pools, kvs)
    assert kvs[0].status() == flags


@pytest.mark.parametrize("t", TYPES)
def test_keep_long_lists(gpu, t):
    rng = np.random.default_rng(3)
    new = [500, 130, 64, 65]
    keeps = [sorted(rng.choice(n, m, replace=False).tolist()) for n, m in zip(new, (300, 129, 64, 63))]
    _keep_case(gpu, t, 64, 1, 16, 1, new, [n + 3 for n in new], keeps)


def test_keep_in_many_caches(gpu):
    _keep_case(gpu, F16, 64, 1, 16, 70, [5], [9], [[0, 2, 4]])


@pytest.mark.parametrize("given,moved", [([0, 2, 2, 4], [0, 2]), ([0, 3, 1], [0, 3]), ([0, 9], [0]), ([-1, 2], []), ([2, 2 ** 31 - 1], [2]), ([0, -2 ** 31], [0])])
def test_keep_ends_where_a_list_does_not_ascend(gpu, given, moved):
    _keep_case(gpu, Q8_0, 64, 2, 16, 2, [9, 4], [20, 10], [moved, [1, 3]], most=6, given=[given, [1, 3]], flags=gpu.PAGED_BAD_BATCH)


def test_keep_behind_64_entries_that_ascend(gpu):
    _keep_case(gpu, F16, 64, 1, 16, 1, [200], [210], [list(range(1, 65))], most=80, given=[list(range(1, 65)) + [64, 90]], flags=gpu.PAGED_BAD_BATCH)


def test_keep_of_bad_counts_moves_nothing(gpu):
    G = gpu
    pools, kvs, caches = _caches(G, F16, 1, 64, 16, 4, 1)
    B = G.Buffer.from_array
    off, table = B(np.array([0, 5, 8, 10, 12], np.int32)), B(np.array([[0], [1], [2], [3]], np.int32))
    batch = G.PagedBatch(4, 12, B(np.array([9, 7, 100, 1], np.int32)), table, 1, 16, q_off=off)
    G.paged_keep(caches, batch, B(np.array([6, -1, 2, 1], np.int32)), B(np.tile(np.array([1, 2, 3, 4, 5, 6], np.int32), 4)), 6)
    _same(pools, kvs)
    assert kvs[0].status() == G.PAGED_BAD_BATCH


def test_keep_leaves_rows_of_bad_pages(gpu):
    G = gpu
    pools, kvs, caches = _caches(G, F16, 2, 64, 16, 4, 2)
    B = G.Buffer.from_array
    batch = G.PagedBatch(1, 20, B(np.array([40], np.int32)), B(np.array([[0, 3, 4]], np.int32)), 3, 48, q_off=B(np.array([0, 20], np.int32)))
    G.paged_keep(caches, batch, B(np.array([3], np.int32)), B(np.array([[2, 5, 15]], np.int32)), 3)   # slots 22, 25, 35 (page 4: none)
    for p in pools:
        _moved(p, [0, 3, 0], 20, [2, 5])
    _same(pools, kvs)
    assert kvs[0].status() == G.PAGED_BAD_PAGE


# -------------------------------------------------------- a run of them together
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("window", [0, 24])
def test_drafts_verified_step_by_step(gpu, t, window):
    """Steps of drafts of changing shape: what the caches hold of each sequence is what
    storing the confirmed tokens one behind the other would have given, bit for bit,
    and a confirmed token's attention is that of the sequence up to it."""
    G, hd, n_head, n_kv, page, layers, n_seq, vocab = gpu, 64, 4, 2, 16, 3, 3, 3
    rng, B = np.random.default_rng(30), gpu.Buffer.from_array
    n_pages, stride = 40, 10
    table = np.arange(n_seq * stride, dtype=np.int32).reshape(n_seq, stride)[:, ::-1].copy()
    made = [[G.PagedKV(t, n_kv, hd, page, n_pages) for _ in range(layers)] for _ in range(2)]
    drafted, plain = made
    caches, rope, table_dev = G.PagedCaches(drafted), G.Rope(hd, 1e4), B(table)
    # a token's rows in layer l depend on the token and its position alone
    emb = rng.standard_normal((layers, 2, vocab, n_kv, hd)).astype(np.float32)
    q_of = rng.standard_normal((vocab, n_head, hd)).astype(np.float32)
    lens, last, held = [0] * n_seq, [0] * n_seq, [[] for _ in range(n_seq)]
    for step in range(6):
        new = [int(x) for x in rng.integers(1, [3, 20, 12, 40, 7, 30][step], n_seq)]
        off = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        parents = [random_parents(rng, n, 0.05) for n in new]
        tokens = [[last[s]] + rng.integers(0, vocab, n - 1).tolist() for s, n in enumerate(new)]
        choice = [rng.integers(0, vocab, n).tolist() for n in new]
        flat, n_tok, words = np.concatenate(tokens), int(off[-1]), -(-max(new) // 32)
        full = [n + m for n, m in zip(lens, new)]
        par, tok, cho = (B(np.asarray(sum(x, []), np.int32)) for x in (parents, tokens, choice))
        batch = G.PagedBatch(n_seq, n_tok, B(np.asarray(full, np.int32)), table_dev, stride, stride * page, q_off=B(off))
        mask, depth = G.Buffer(4 * n_tok * words), G.Buffer(4 * n_tok)
        tree, q = G.PagedTree(words, mask, depth), B(q_of[flat])
        G.paged_tree_build(batch, par, words, mask, depth)
        outs = []
        for layer, kv in enumerate(drafted):
            turned, out = G.Buffer(q.nbytes), G.Buffer(q.nbytes)
            G.paged_append_tree(kv, batch, tree, B(emb[layer, 0][flat]), B(emb[layer, 1][flat]), q=q, q_out=turned, n_head=n_head, rope=rope)
            G.paged_attn_tree(kv, batch, tree, turned, n_head, out, scale=0.125, window=window)
            outs.append(out.download(np.float32, (n_tok, n_head, hd)))
        n_keep, keep, nxt, out_len = (G.Buffer(4 * m) for m in (n_seq, n_seq * 8, n_seq, n_seq))
        G.paged_tree_accept(batch, par, tok, cho, 8, n_keep, keep, next_out=nxt, len_out=out_len)
        G.paged_keep(caches, batch, n_keep, keep, 8)
        paths = [walk(p, x, c, 8) for p, x, c in zip(parents, tokens, choice)]
        assert keep.download(np.int32, (n_seq, 8)).tolist() == [p + [-1] * (8 - len(p)) for p, _ in paths]
        # the same tokens, one behind the other
        kept = [len(p) for p, _ in paths]
        line = np.concatenate([np.asarray(tokens[s])[paths[s][0]] for s in range(n_seq)])
        koff = np.concatenate([[0], np.cumsum(kept)]).astype(np.int32)
        lens = [n + m for n, m in zip(lens, kept)]
        pb = G.PagedBatch(n_seq, len(line), B(np.asarray(lens, np.int32)), table_dev, stride, stride * page, q_off=B(koff))
        for layer, kv in enumerate(plain):
            turned, out = G.Buffer(4 * len(line) * n_head * hd), G.Buffer(4 * len(line) * n_head * hd)
            G.paged_append(kv, pb, B(emb[layer, 0][line]), B(emb[layer, 1][line]), q=B(q_of[line]), q_out=turned, n_head=n_head, rope=rope)
            G.paged_attn(kv, pb, turned, n_head, out, scale=0.125, window=window)
            want = out.download(np.float32, (len(line), n_head, hd))
            for s in range(n_seq):
                got = outs[layer][off[s] + np.asarray(paths[s][0])]
                # each within 2 d of an average of values of unit size (paged_util.attend): d below 8 (2^-21 + 64 2^-24)
                # where |q| |k| / 8 stays below 8 (64 products of unit size: 5), so 2^-13.8 each
                assert np.abs(got - want[koff[s]:koff[s + 1]]).max() <= 2.0 ** -12
        assert out_len.download(np.int32, (n_seq,)).tolist() == lens
        last = nxt.download(np.int32, (n_seq,)).tolist()
        assert last == [x for _, x in paths]
        # every row that the caches hold
        rb = G.PagedBatch(n_seq, sum(lens), B(np.asarray(lens, np.int32)), table_dev, stride, stride * page,
                          q_off=B(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)))
        for a, b in zip(drafted, plain):
            rows = []
            for kv in (a, b):
                k, v = G.Buffer(4 * sum(lens) * n_kv * hd), G.Buffer(4 * sum(lens) * n_kv * hd)
                G.paged_read(kv, rb, k, v)
                rows.append([x.download(np.float32, (sum(lens), n_kv, hd)) for x in (k, v)])
            assert np.array_equal(rows[0][0], rows[1][0]) and np.array_equal(rows[0][1], rows[1][1])
    assert drafted[0].status() == 0
