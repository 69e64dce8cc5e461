"""Draft trees over the paged KV cache at the shapes where their kernels change
what they do: query groups of all sizes, masks too long to be held, pieces longer
than the page ids held at once, all of prefix, window and cap together, pools past
4 GiB, workspaces shared by captured graphs."""
import numpy as np
import pytest

import paged_util as U
from paged_util import F16, Q4_0, Q8_0
from tree_util import TreeCase, ancestry, pack, random_parents

pytestmark = pytest.mark.gpu
TYPES = [F16, Q8_0, Q4_0]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd,n_head,n_kv", [(64, 3, 1), (64, 34, 2), (64, 128, 1), (128, 5, 1), (128, 12, 1), (128, 65, 1), (128, 128, 1), (256, 3, 1),
                                            (256, 40, 1), (256, 65, 1), (256, 128, 1), (512, 7, 1), (512, 20, 1), (512, 33, 1), (512, 64, 1)])
@pytest.mark.parametrize("new", [[1, 1], [5], [9, 2]])
def test_groups_of_query_heads(gpu, t, hd, n_head, n_kv, new):
    TreeCase(gpu, t, n_head, n_kv, hd, 16, [n + 45 for n in new], new, seed=n_head).check()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd,n_head", [(64, 1), (128, 2), (256, 1), (512, 1)])
@pytest.mark.parametrize("n,words", [(130, 8), (40, 32)])
def test_masks_of_more_words_than_are_held(gpu, t, hd, n_head, n, words):
    TreeCase(gpu, t, n_head, 1, hd, 16, [n + 30, 20], [n, 3], words=words, seed=words).check()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("new", [[5], [20, 7], [70]])
@pytest.mark.parametrize("window", [0, 30])
def test_prefix_window_and_cap_together(gpu, t, hd, new, window):
    c = TreeCase(gpu, t, 2, 1, hd, 16, [n + 25 + 9 * i for i, n in enumerate(new)], new, n_prefix=45, seed=window + hd)
    c.check(cap=20.0, window=window)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("first", [0, 1, 31, 32, 33, 63, 64, 127, 128])
def test_where_tiles_of_positions_end(gpu, t, hd, first):
    TreeCase(gpu, t, 2, 1, hd, 16, [first + 18, first + 1], [18, 1], seed=first).check()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd,page", [(64, 16), (128, 64), (256, 48), (512, 32)])
@pytest.mark.parametrize("new", [3, 19])
def test_pieces_longer_than_the_page_ids_held(gpu, t, hd, page, new):
    """As many copies of one sequence as give a workgroup most of one: a piece of over 2000 positions."""
    G = gpu
    copies, n_kv = 120, 2
    c = TreeCase(G, t, n_kv, n_kv, hd, page, [2600], [new], seed=hd)
    want, tol = c.expect(hd ** -0.5)
    B = G.Buffer.from_array
    off = B(np.arange(0, new * copies + 1, new, dtype=np.int32))
    batch = G.PagedBatch(copies, new * copies, B(np.full(copies, 2600, np.int32)), B(np.tile(c.table, (copies, 1))), c.stride, 2600, q_off=off)
    tree = G.PagedTree(c.words, B(np.tile(pack(c.sets, c.words), (copies, 1))), B(np.tile(np.asarray(c.depths, np.int32), copies)))
    out = G.Buffer(copies * new * n_kv * hd * 4)
    G.paged_attn_tree(c.kv, batch, tree, B(np.tile(c.q, (copies, 1, 1))), n_kv, out, scale=hd ** -0.5)
    got = out.download(np.float32, (copies, new, n_kv, hd))
    assert (np.abs(got - want) <= tol).all()
    assert c.kv.status() == 0


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [128, 256, 512])
@pytest.mark.parametrize("new", [[8], [44]])
def test_slots_that_a_row_does_not_attend_may_hold_anything(gpu, t, hd, new):
    c = TreeCase(gpu, t, 2, 1, hd, 16, [n + 20 for n in new], new, seed=23)
    clean = c.attn(0.125)
    slot, row = c.lens[0] - new[0] + 2, U.row_bytes(t, hd)
    page, s = c.table[0, slot // 16], slot % 16
    at, n = (s * row, row) if t == F16 else (16 * row + s * (hd // 16), hd // 16)
    for kind in (0x7c00, 0xfc00, 0x7e00):                    # infinities, NaN: of values, or of scales
        for raw in (c.pool.k, c.pool.v):
            raw[page, at:at + n] = np.full(n // 2, kind, np.uint16).view(np.uint8)
        c.kv.k.upload(c.pool.k)
        c.kv.v.upload(c.pool.v)
        got = c.attn(0.125)
        reads = np.array([2 in s for s in c.sets])
        assert reads.any() and not reads.all()
        assert not np.isfinite(got[reads]).all(-1).any()
        assert np.array_equal(got[~reads], clean[~reads])


@pytest.mark.parametrize("t,hd,page", [(F16, 128, 64), (Q8_0, 256, 48)])
@pytest.mark.parametrize("new", [[7], [30]])
def test_offsets_past_32_bits(gpu, t, hd, page, new):
    """Pages more than 4 GiB into the pools: attended, and rows moved among them."""
    G = gpu
    n_kv, pb = 4, U.page_bytes(t, 4, hd, page)
    n_pages = (9 << 30) // 2 // pb
    kv = G.PagedKV(t, n_kv, hd, page, n_pages)
    c = TreeCase(G, t, 8, n_kv, hd, page, [page + 20 + new[0]], new, seed=24)
    table = np.full_like(c.table, -7)
    L = G.lib()

    def row(buf, i):
        got = np.zeros(pb, np.uint8)
        G.check(L.g4h_memcpy_d2h(got.ctypes.data, buf.ptr + int(table[0, i]) * pb, pb, None))
        G.synchronize()
        return got

    used = -(-c.lens[0] // page)
    for i in range(used):
        table[0, i] = n_pages - 1 - i
        for buf, rows in ((kv.k, c.pool.k), (kv.v, c.pool.v)):
            x = np.ascontiguousarray(rows[c.table[0, i]])
            G.check(L.g4h_memcpy_h2d(buf.ptr + int(table[0, i]) * pb, x.ctypes.data, pb, None))
            G.synchronize()
    small = c.kv
    c.kv = kv
    c.d["table"].upload(table)
    c.check()
    keep = [0, 2, 3, new[0] - 1]
    B = G.Buffer.from_array
    n_keep, keeps = B(np.array([len(keep)], np.int32)), B(np.array([keep], np.int32))
    G.paged_keep(G.PagedCaches([kv]), c.batch, n_keep, keeps, len(keep))
    c.d["table"].upload(c.table)
    G.paged_keep(G.PagedCaches([small]), c.batch, n_keep, keeps, len(keep))
    for big, few in ((kv.k, small.k), (kv.v, small.v)):
        want = few.download(np.uint8, c.pool.k.shape)
        for i in range(used):
            assert np.array_equal(row(big, i), want[c.table[0, i]]), i
    # a fresh page far from the parent's
    c.d["table"].upload(table)
    fork = G.PagedBatch(1, 0, B(np.array(c.lens, np.int32)), c.d["table"], c.stride, c.max_len)
    lens, out = G.Buffer(4), G.Buffer(4 * (used + 1))
    G.paged_fork(G.PagedCaches([kv]), fork, 1, B(np.array([0], np.int32)), B(np.array([5], np.int32)), lens, out, used + 1)
    got = out.download(np.int32, (used + 1,))
    part = c.lens[0] % page
    assert part and got[:used].tolist() == table[0, :used - 1].tolist() + [5] and lens.download(np.int32, (1,))[0] == c.lens[0]
    old = row(kv.k, used - 1)
    table[0, used - 1] = 5
    new_row, n = row(kv.k, used - 1), U.row_bytes(t, hd)
    for h in range(n_kv):
        assert np.array_equal(new_row[h * page * n:(h * page + part) * n], old[h * page * n:(h * page + part) * n])


@pytest.mark.parametrize("t", TYPES)
def test_two_graphs_share_a_workspace(gpu, t):
    """One after the other on a stream, in any order, with eager calls between them."""
    G = gpu
    cases = [TreeCase(G, t, 4, 2, 128, 16, [600, 90], [6, 9], seed=25), TreeCase(G, t, 4, 2, 128, 16, [900], [40], n_prefix=70, seed=26)]
    s = G.Stream()
    ws = G.Buffer(max(G.paged_attn_tree_workspace_bytes(c.kv, c.batch, 4) for c in cases))
    outs = [G.Buffer(c.n_tok * 4 * 128 * 4) for c in cases]
    run = [lambda c=c, o=o: G.paged_attn_tree(c.kv, c.batch, c.tree, c.d["q"], 4, o, scale=0.1, ws=ws, stream=s.ptr) for c, o in zip(cases, outs)]
    graphs = []
    for r in run:
        r()
        s.synchronize()
        graphs.append(G.Graph(s.ptr, r))
    want = [c.expect(0.1) for c in cases]
    for order in ([0, 1], [1, 0], [0, 0, 1], [1]):
        for o, c in zip(outs, cases):
            o.upload(np.full((c.n_tok, 4, 128), 3.0, np.float32), s.ptr)
        for i in order:
            graphs[i].launch(s.ptr)
        run[order[0]]()
        s.synchronize()
        for i in set(order):
            got = outs[i].download(np.float32, want[i][0].shape)
            assert (np.abs(got - want[i][0]) <= want[i][1]).all(), (order, i)


@pytest.mark.parametrize("t", TYPES)
def test_a_draft_step_replayed(gpu, t):
    """Masks, rotation, attention, the walk and the rows moved, in one graph, replayed over other trees."""
    G = gpu
    n, hd, n_kv, n_head, page, first = [11, 3, 24], 128, 2, 4, 16, 50
    c = TreeCase(G, t, n_head, n_kv, hd, page, [first + x for x in n], n, seed=27)
    B, n_tok, rng = G.Buffer.from_array, sum(n), np.random.default_rng(28)
    k, v = (rng.standard_normal((n_tok, n_kv, hd)).astype(np.float32) for _ in range(2))
    kb, vb, q = B(k), B(v), B(c.q)
    par, tok, cho = (B(np.zeros(n_tok, np.int32)) for _ in range(3))
    mask, depth, flags = G.Buffer(4 * n_tok), G.Buffer(4 * n_tok), B(np.zeros(1, np.int32))
    nk, keep, nxt, lout = G.Buffer(12), G.Buffer(12 * 8), G.Buffer(12), G.Buffer(12)
    q_out, out, s = G.Buffer(c.q.nbytes), G.Buffer(c.q.nbytes), G.Stream()
    ws = G.Buffer(max(16, G.paged_attn_tree_workspace_bytes(c.kv, c.batch, n_head)))
    rope, tree, caches = G.Rope(hd, 1e4, False, None), G.PagedTree(1, mask, depth), G.PagedCaches([c.kv])

    def step():
        G.paged_tree_build(c.batch, par, 1, mask, depth, flags, stream=s.ptr)
        G.paged_append_tree(c.kv, c.batch, tree, kb, vb, q=q, q_out=q_out, n_head=n_head, rope=rope, stream=s.ptr)
        G.paged_attn_tree(c.kv, c.batch, tree, q_out, n_head, out, scale=0.1, ws=ws, stream=s.ptr)
        G.paged_tree_accept(c.batch, par, tok, cho, 8, nk, keep, nxt, lout, flags, stream=s.ptr)
        G.paged_keep(caches, c.batch, nk, keep, 8, stream=s.ptr)

    def results():
        s.synchronize()
        return [x.download(np.uint8, (x.nbytes,)) for x in (mask, depth, out, nk, keep, nxt, lout, c.kv.k, c.kv.v)]

    clean = c.kv.k.download(np.uint8, c.pool.k.shape), c.kv.v.download(np.uint8, c.pool.v.shape)
    step()                                                   # parents of 0: of the first tokens, flagged and as if -1
    results()
    assert flags.download(np.int32, (1,))[0] == G.PAGED_BAD_BATCH
    flags.upload(np.zeros(1, np.int32))
    g = G.Graph(s.ptr, step)
    for _ in range(4):
        trees = [random_parents(rng, x) for x in n]
        par.upload(np.array(sum(trees, []), np.int32), s.ptr)
        tok.upload(rng.integers(0, 3, n_tok).astype(np.int32), s.ptr)
        cho.upload(rng.integers(0, 3, n_tok).astype(np.int32), s.ptr)
        got = []
        for run in (lambda: g.launch(s.ptr), step, lambda: g.launch(s.ptr)):
            c.kv.k.upload(clean[0], s.ptr)
            c.kv.v.upload(clean[1], s.ptr)
            run()
            got.append(results())
        for other in got[1:]:
            assert all(np.array_equal(a, b) for a, b in zip(got[0], other))
        sets, depths = (sum((ancestry(p)[i] for p in trees), []) for i in (0, 1))
        assert np.array_equal(got[0][0].view(np.uint32), pack(sets, 1)[:, 0]) and got[0][1].view(np.int32).tolist() == depths
    assert flags.download(np.int32, (1,))[0] == 0 and c.kv.status() == 0
