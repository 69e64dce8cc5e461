"""Beam search's selection against float64 (tests/tree_util.py), the carried-over
beams' tables and pages, and a search with both over the paged KV cache."""
import numpy as np
import pytest

from paged_util import F16, Q4_0, Q8_0
from test_gpu_tree import _caches, _rows, _same
from tree_util import select

pytestmark = pytest.mark.gpu
TYPES = [F16, Q8_0, Q4_0]


def _select(G, x, score, n_beam, n_out, ended=None, stride=0, shift=0, stream=None, ws=None):
    rows, vocab = x.shape
    g = rows // n_beam
    B = G.Buffer.from_array
    if stride or shift:
        wide = np.full((rows, stride or vocab), 1e30, np.float32)
        wide[:, :vocab] = x
        x = np.concatenate([np.full(shift, np.nan, np.float32), wide.reshape(-1)])
    xd = B(np.ascontiguousarray(x, np.float32))
    out = [G.Buffer.from_array(np.full((g, n_out), 99, np.int32)) for _ in range(3)]
    G.beam_select(xd.ptr + 4 * shift, g, n_beam, vocab, B(np.asarray(score, np.float32)), n_out, *out,
                  ended=B(np.asarray(ended, np.int32)) if ended is not None else None, stride=stride, ws=ws, stream=stream)
    return out[0].download(np.float32, (g, n_out)), *(o.download(np.int32, (g, n_out)) for o in out[1:])


def _check(G, x, score, n_beam, n_out, **more):
    got = _select(G, x, score, n_beam, n_out, **more)
    want = select(x, score, n_beam, n_out, more.get("ended"))
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])
    live = want[1] >= 0
    assert (got[0][~live] == -np.inf).all()
    # the normaliser: exponentials of arguments rounded to fp32 (2^-24 of up to 40 each, 2^-22 of their own), sums of
    # up to 32 and 256 of them in fp32 (2^-24 each, of positive terms: 2^-17 at worst), and the score rounded to fp32
    tol = 40 * 2.0 ** -24 + 2.0 ** -22 + 2.0 ** -17 + np.abs(want[0][live]) * 2.0 ** -24
    assert (np.abs(got[0][live] - want[0][live]) <= tol).all()
    return got


@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 65, 1000, 2047, 2048, 2049, 8192, 8193, 50001])
@pytest.mark.parametrize("n_group,n_beam,n_out", [(1, 1, 1), (1, 4, 8), (3, 5, 5), (2, 64, 64), (1, 3, 64)])
def test_select(gpu, vocab, n_group, n_beam, n_out):
    rng = np.random.default_rng(vocab + n_beam)
    x = (rng.standard_normal((n_group * n_beam, vocab)) * 3).astype(np.float32)
    _check(gpu, x, -4 * rng.random(n_group * n_beam, np.float32), n_beam, n_out)


@pytest.mark.parametrize("rows,n_beam,vocab,n_out", [(96, 8, 50001, 16), (600, 4, 8193, 4), (700, 2, 1000, 7), (24, 8, 262144, 16), (1024, 64, 3001, 64)])
def test_select_of_many_rows(gpu, rows, n_beam, vocab, n_out):
    rng = np.random.default_rng(rows)
    x = rng.standard_normal((rows, vocab), np.float32) * np.float32(2.5)
    _check(gpu, x, -4 * rng.random(rows, np.float32), n_beam, n_out)


def test_select_of_a_long_row(gpu):
    # more chunks than a wave has lanes
    rng = np.random.default_rng(1)
    x = rng.standard_normal((2, 1 << 20), np.float32) * np.float32(2)
    _check(gpu, x, [-1.0, -1.25], 2, 40)


@pytest.mark.parametrize("order", ["rising", "falling", "nothing first", "level", "steps"])
@pytest.mark.parametrize("rows,vocab,n_out", [(300, 20011, 7), (512, 16385, 64), (1024, 12289, 1)])
def test_rows_of_several_chunks(gpu, order, rows, vocab, n_out):
    # many rows: a workgroup looks through several chunks of one, its bound rising as it goes
    rng = np.random.default_rng(rows)
    x = rng.standard_normal((rows, vocab), np.float32)
    if order in ("rising", "falling"):
        x.sort(axis=1)
    if order == "falling":
        x = x[:, ::-1]
    if order == "nothing first":
        x[:, :9000] = -np.inf
        x[::2, :4500] = np.nan
        x[::3, 9000:12288] = -np.inf
    if order == "level":
        x[:] = 0.5
        x[::2, 4096:] = 0.75                                 # above what the first chunk left, all of it
    if order == "steps":
        x = np.floor(np.arange(vocab) / 1000 + x).astype(np.float32) / 4
    # beams far enough apart that no two rows' normalisers decide
    _check(gpu, np.ascontiguousarray(x), np.tile([0.0, -60.0, -120.0, -180.0], rows // 4), 4, n_out)


@pytest.mark.parametrize("stride,shift", [(1009, 0), (1001, 1), (0, 3), (1003, 2)])
def test_rows_of_any_stride_and_alignment(gpu, stride, shift):
    rng = np.random.default_rng(stride + shift)
    x = rng.standard_normal((12, 1001), np.float32)
    _check(gpu, x, -rng.random(12, np.float32), 4, 6, stride=stride, shift=shift)


@pytest.mark.parametrize("vocab", [500, 9000, 40000])
@pytest.mark.parametrize("levels", [1, 2, 7])
@pytest.mark.parametrize("rows", [4, 512])
def test_equal_logits_go_by_token(gpu, vocab, levels, rows):
    if rows * vocab > 1 << 23:
        pytest.skip("no other path than the smaller ones")
    rng = np.random.default_rng(levels)
    x = rng.integers(0, levels, (rows, vocab)).astype(np.float32)
    x[0, ::3] *= -1                                          # -0 is 0
    # beams a whole unit apart or more: their order does not hang on a normaliser's last bits
    _check(gpu, x, -40.0 * np.arange(rows), 4, 33)


def test_equal_rows_go_by_row(gpu):
    rng = np.random.default_rng(2)
    x = np.repeat(rng.standard_normal((1, 5001), np.float32), 8, 0)
    got = _check(gpu, x, np.full(8, -2.0), 8, 20)
    assert got[1].tolist() == [[0, 1, 2, 3, 4, 5, 6, 7] * 2 + [0, 1, 2, 3]]
    # at other alignments and strides too
    _check(gpu, x, np.full(8, -2.0), 8, 20, stride=5003, shift=1)


def test_rows_and_tokens_that_are_never_selected(gpu):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((16, 3000), np.float32)
    score = -rng.random(16).astype(np.float32)
    x[1, 77], x[2, 5], x[3], x[4, 10:] = np.nan, np.inf, -np.inf, -np.inf
    x[5, :2999] = -np.inf
    score[6], score[7] = -np.inf, np.nan
    x[8:, 7] = np.nan                                        # the last group's all
    for n_out in (3, 60):
        _check(gpu, x, score, 8, n_out)
    _check(gpu, np.full((4, 100), -np.inf, np.float32), np.zeros(4), 4, 5)
    _check(gpu, np.full((4, 9000), np.nan, np.float32), np.zeros(4), 2, 5)


@pytest.mark.parametrize("size", [1e-30, 1e-3, 80.0, 1e4, 3e38])
def test_logits_of_any_size(gpu, size):
    rng = np.random.default_rng(4)
    x = (rng.uniform(-1, 1, (6, 3000)) * size).astype(np.float32)
    # a beam a group where the spread leaves scores apart by less than their rounding
    got = _select(gpu, x, np.zeros(6), 1, 9)
    want = select(x, np.zeros(6), 1, 9)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])
    assert (np.abs(got[0] - want[0]) <= 40 * 2.0 ** -24 + 2.0 ** -22 + 2.0 ** -17 + np.abs(want[0]) * 2.0 ** -23).all()


def test_scores_that_are_infinite_or_large(gpu):
    x = np.random.default_rng(5).standard_normal((4, 100)).astype(np.float32)
    got = _select(gpu, x, np.array([0, np.inf, -3e38, 3e38]), 4, 6)
    assert (got[0][0] == np.inf).all() and (got[1] == 1).all() and got[2][0].tolist() == select(x[1:2], [0.0], 1, 6)[2][0].tolist()


@pytest.mark.parametrize("n_out", [2, 4, 16])
def test_ended_rows(gpu, n_out):
    rng = np.random.default_rng(6)
    x = rng.standard_normal((12, 700), np.float32)
    ended = np.array([0, 1, 0, 2, 1, 1, 1, 1, 0, 0, -1, 0])
    score = -3 * rng.random(12).astype(np.float32)
    score[5], score[6] = -np.inf, np.nan
    score[1] = 2.0                                           # the best of its group
    x[3], x[10] = np.nan, np.inf                             # not read
    got = _check(gpu, x, score, 4, n_out, ended=ended)
    assert got[2][0, 0] == -1 and got[1][0, 0] == 1 and got[0][0, 0] == 2.0


def test_the_first_step_has_one_beam(gpu):
    rng = np.random.default_rng(7)
    x = np.repeat(rng.standard_normal((3, 2000), np.float32), 4, 0)
    got = _check(gpu, x, np.tile([0, -np.inf, -np.inf, -np.inf], 3), 4, 4)
    assert (got[1] == np.arange(0, 12, 4)[:, None]).all()


def test_scores_in_place(gpu):
    G = gpu
    rng = np.random.default_rng(8)
    x, score = rng.standard_normal((40, 300), np.float32), -rng.random(40, np.float32)
    B = G.Buffer.from_array
    s, row, token = B(score), G.Buffer(160), G.Buffer(160)
    G.beam_select(B(x), 10, 4, 300, s, 4, s, row, token)
    want = _select(G, x, score, 4, 4)
    assert np.array_equal(s.download(np.float32, (10, 4)), want[0]) and np.array_equal(row.download(np.int32, (10, 4)), want[1])


def test_no_groups(gpu):
    G = gpu
    assert G.beam_workspace_bytes(0, 4, 100, 4) == 0
    G.beam_select(None, 0, 4, 100, None, 4, None, None, None)


def test_graph_replays_and_repeats(gpu):
    G = gpu
    rng, B = np.random.default_rng(9), G.Buffer.from_array
    x, score, s = B(np.zeros((32, 20011), np.float32)), B(np.zeros(32, np.float32)), G.Stream()
    out = [G.Buffer(4 * 4 * 16) for _ in range(3)]
    ws = B(np.full(G.beam_workspace_bytes(4, 8, 20011, 16), 0xff, np.uint8))
    g = G.Graph(s.ptr, lambda: G.beam_select(x, 4, 8, 20011, score, 16, *out, ws=ws, stream=s.ptr))
    for _ in range(4):
        xa, sa = rng.standard_normal((32, 20011), np.float32) * np.float32(3), -rng.random(32, np.float32)
        x.upload(xa, s.ptr)
        score.upload(sa, s.ptr)
        first = None
        for _ in range(2):
            g.launch(s.ptr)
            s.synchronize()
            got = [o.download(t, (4, 16)) for o, t in zip(out, (np.float32, np.int32, np.int32))]
            assert first is None or all(np.array_equal(a, b) for a, b in zip(first, got))
            first = got
        want = _check(G, xa, sa, 8, 16)
        assert all(np.array_equal(a, b) for a, b in zip(first, want))


# ------------------------------------------------------------------------- fork
def _fork_case(G, t, hd, n_kv, page, n_cache, lens, parent, out_stride=None, fresh=None, flags=0, bad=(), max_len=None):
    """bad: rows that the call leaves out.  Page ids: the sequences' own, then the fresh ones."""
    rng = np.random.default_rng(11)
    need = [-(-n // page) for n in lens]
    ids = rng.permutation(sum(need) + len(parent) + 1)
    stride = max(need + [1]) + 1
    table = np.full((len(lens), stride), -5, np.int32)
    for i, n in enumerate(need):
        table[i, :n] = ids[sum(need[:i]):sum(need[:i]) + n]
    fresh = ids[sum(need):sum(need) + len(parent)].astype(np.int32) if fresh is None else fresh(table)
    pools, kvs, caches = _caches(G, t, n_kv, hd, page, len(ids), n_cache, seed=hd)
    B = G.Buffer.from_array
    out_stride = stride if out_stride is None else out_stride
    batch = G.PagedBatch(len(lens), 0, B(np.asarray(lens, np.int32)), B(table), stride, max_len or max(lens + [1]))
    tout, lout = np.full((len(parent), out_stride), -9, np.int32), np.full(len(parent), 77, np.int32)
    td, ld = B(tout), B(lout)
    G.paged_fork(caches, batch, len(parent), B(np.asarray(parent, np.int32)), B(fresh), ld, td, out_stride)
    old = [(p.k.copy(), p.v.copy()) for p in pools]
    for i, up in enumerate(parent):
        if i in bad or up < 0:
            lout[i] = 0
            continue
        whole, part = divmod(lens[up], page)
        lout[i] = lens[up]
        tout[i, :whole] = table[up, :whole]
        if whole < out_stride:
            tout[i, whole] = fresh[i]
        if part and 0 <= fresh[i] < len(ids):
            for p, o in zip(pools, old):
                for raw, was in ((p.k, o[0]), (p.v, o[1])):
                    for x, y in zip(_rows(p, raw), _rows(p, was)):
                        x[fresh[i], :, :part] = y[table[up, whole], :, :part]
    assert np.array_equal(td.download(np.int32, tout.shape), tout) and ld.download(np.int32, lout.shape).tolist() == lout.tolist()
    _same(pools, kvs)
    assert kvs[0].status() == flags


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd,n_kv,page", [(64, 3, 16), (128, 8, 48), (256, 1, 32), (512, 2, 16)])
@pytest.mark.parametrize("n_cache", [1, 3])
def test_fork(gpu, t, hd, n_kv, page, n_cache):
    _fork_case(gpu, t, hd, n_kv, page, n_cache, [0, 1, page - 1, page, page + 1, 3 * page, 3 * page + 7], [6, 6, 5, 0, 1, 2, 3, 4, 6, -1, 2])


def test_fork_of_large_pages_and_many_caches(gpu):
    _fork_case(gpu, F16, 128, 2, 1024, 2, [1500, 700], [1, 0, 0])
    _fork_case(gpu, Q4_0, 64, 1, 16, 70, [9], [0, 0])


def test_fork_goes_on_in_the_parents_page(gpu):
    def fresh(table):
        return np.array([table[1, 1], 9, 8], np.int32)
    # pages 0 .. 8 of two sequences of 3 and 3, then others
    G = gpu
    pools, kvs, caches = _caches(G, Q8_0, 2, 64, 16, 12, 2)
    B = G.Buffer.from_array
    table = np.array([[0, 1, 2], [3, 4, 5]], np.int32)
    batch = G.PagedBatch(2, 0, B(np.array([20, 25], np.int32)), B(table), 3, 48)
    lout, tout = G.Buffer(12), B(np.full((3, 3), -1, np.int32))
    G.paged_fork(caches, batch, 3, B(np.array([1, 1, 0], np.int32)), B(fresh(table)), lout, tout, 3)
    for p in pools:
        for raw in (p.k, p.v):
            for x in _rows(p, raw):
                x[9, :, :9], x[8, :, :4] = x[4, :, :9].copy(), x[1, :, :4].copy()
    _same(pools, kvs)
    assert tout.download(np.int32, (3, 3)).tolist() == [[3, 4, -1], [3, 9, -1], [0, 8, -1]]


def test_fork_of_bad_rows(gpu):
    bad = gpu.PAGED_BAD_BATCH
    _fork_case(gpu, F16, 64, 2, 16, 1, [20, 40, 33], [3, 0, -2, 2 ** 31 - 1, -1, 1], flags=bad, bad=(0, 2, 3))
    _fork_case(gpu, F16, 64, 2, 16, 1, [20, 40, 33], [0, 1, 2], out_stride=2, flags=bad, bad=(1, 2))
    _fork_case(gpu, F16, 64, 2, 16, 1, [20, 40, 32], [0, 1, 2], max_len=35, flags=bad, bad=(1,))
    _fork_case(gpu, F16, 64, 2, 16, 1, [20, 32], [0, 1, 1], fresh=lambda table: np.array([99, -4, 99], np.int32), flags=gpu.PAGED_BAD_PAGE)


def test_fork_of_a_bad_parents_page(gpu):
    G = gpu
    pools, kvs, caches = _caches(G, F16, 1, 64, 16, 4, 1)
    B = G.Buffer.from_array
    batch = G.PagedBatch(2, 0, B(np.array([20, 5], np.int32)), B(np.array([[0, 7], [-1, 0]], np.int32)), 2, 32)
    lout, tout = G.Buffer(8), G.Buffer(16)
    G.paged_fork(caches, batch, 2, B(np.array([0, 1], np.int32)), B(np.array([2, 3], np.int32)), lout, tout, 2)
    _same(pools, kvs)
    assert kvs[0].status() == G.PAGED_BAD_PAGE and lout.download(np.int32, (2,)).tolist() == [20, 5]


def test_fork_without_tables(gpu):
    G = gpu
    pools, kvs, caches = _caches(G, F16, 1, 64, 16, 4, 2)
    B = G.Buffer.from_array
    batch = G.PagedBatch(1, 0, B(np.array([5], np.int32)), B(np.array([[1]], np.int32)), 1, 16)
    G.paged_fork(caches, batch, 1, B(np.array([0], np.int32)), B(np.array([2], np.int32)), None, None, 1)
    for p in pools:
        for raw in (p.k, p.v):
            x = _rows(p, raw)[0]
            x[2, :, :5] = x[1, :, :5]
    _same(pools, kvs)


# -------------------------------------------------------- a run of them together
@pytest.mark.parametrize("t", TYPES)
def test_a_search_over_the_paged_cache(gpu, t):
    """Steps of append, attention, selection and fork, the next step's batch made from
    their outputs on the device: every beam's cache holds its own history's rows, and
    its attention is that history's."""
    G, hd, n_head, n_kv, page, layers = gpu, 64, 4, 2, 16, 2
    n_group, n_beam, vocab, steps, stride, prompt = 2, 3, 50, 40, 5, 7
    rows, rng, B = n_group * n_beam, np.random.default_rng(12), gpu.Buffer.from_array
    n_pages = rows * stride * 2 + rows * steps
    emb = rng.standard_normal((layers, 2, vocab, n_kv, hd)).astype(np.float32)
    q_of = rng.standard_normal((vocab, n_head, hd)).astype(np.float32)
    head = (rng.standard_normal((n_head * hd, vocab)) * 0.3).astype(np.float32)
    kvs = [G.PagedKV(t, n_kv, hd, page, n_pages) for _ in range(layers)]
    caches, rope = G.PagedCaches(kvs), G.Rope(hd, 1e4)
    free = list(range(n_pages))[::-1]
    # a prompt shared by all beams of a group, each with a page of its own
    table = np.array([[free.pop() for _ in range(1)] + [0] * (stride - 1) for _ in range(rows)], np.int32)
    history = [list(rng.integers(0, vocab, prompt)) if r % n_beam == 0 else None for r in range(rows)]
    history = [list(history[r - r % n_beam]) for r in range(rows)]
    score = np.tile([0.0] + [-np.inf] * (n_beam - 1), n_group).astype(np.float32)
    lens = np.full(rows, prompt, np.int32)
    lens_d, table_d, score_d = B(lens), B(table), B(score)
    off = B((np.arange(rows + 1) * prompt).astype(np.int32))
    first = G.PagedBatch(rows, rows * prompt, lens_d, table_d, stride, stride * page, q_off=off)
    tok = np.concatenate(history)
    for layer, kv in enumerate(kvs):
        G.paged_append(kv, first, B(emb[layer, 0][tok]), B(emb[layer, 1][tok]), rope=rope)
    last = np.array([h[-1] for h in history])
    for step in range(steps):
        batch = G.PagedBatch(rows, rows, lens_d, table_d, stride, stride * page)
        turned, out = G.Buffer(rows * n_head * hd * 4), G.Buffer(rows * n_head * hd * 4)
        x = np.zeros((rows, vocab), np.float32)
        for layer, kv in enumerate(kvs):
            # the last token's rows are in place: appended again, the same
            G.paged_append(kv, batch, B(emb[layer, 0][last]), B(emb[layer, 1][last]), q=B(q_of[last]), q_out=turned, n_head=n_head, rope=rope)
            G.paged_attn(kv, batch, turned, n_head, out, scale=0.125)
            x += out.download(np.float32, (rows, n_head * hd)) @ head
        row_d, token_d, next_score = G.Buffer(rows * 4), G.Buffer(rows * 4), G.Buffer(rows * 4)
        G.beam_select(B(x), n_group, n_beam, vocab, score_d, n_beam, next_score, row_d, token_d)
        want = select(x, score, n_beam, n_beam)
        parent, token = (d.download(np.int32, (rows,)) for d in (row_d, token_d))
        assert np.array_equal(parent, want[1].ravel()) and np.array_equal(token, want[2].ravel())
        score, score_d = next_score.download(np.float32, (rows,)), next_score
        fresh = B(np.array([free.pop() for _ in range(rows)], np.int32))
        lens_o, table_o = G.Buffer(rows * 4), B(np.full((rows, stride), -1, np.int32))
        G.paged_fork(caches, batch, rows, row_d, fresh, lens_o, table_o, stride)
        history = [history[p] + [int(v)] for p, v in zip(parent, token)]
        last = token
        lens = lens_o.download(np.int32, (rows,)) + 1
        lens_d, table_d = B(lens), table_o
    # what the caches hold, against the histories appended to caches of their own
    n = prompt + steps
    batch = G.PagedBatch(rows, rows * (n - 1), B(lens - 1), table_d, stride, stride * page, q_off=B((np.arange(rows + 1) * (n - 1)).astype(np.int32)))
    own_table = np.arange(rows * stride, dtype=np.int32).reshape(rows, stride)
    tok = np.concatenate([h[:-1] for h in history])
    for layer, kv in enumerate(kvs):
        plain = G.PagedKV(t, n_kv, hd, page, rows * stride)
        pb = G.PagedBatch(rows, rows * (n - 1), B(lens - 1), B(own_table), stride, stride * page, q_off=B((np.arange(rows + 1) * (n - 1)).astype(np.int32)))
        G.paged_append(plain, pb, B(emb[layer, 0][tok]), B(emb[layer, 1][tok]), rope=rope)
        got = []
        for which, bt in ((kv, batch), (plain, pb)):
            k, v = (G.Buffer(rows * (n - 1) * n_kv * hd * 4) for _ in range(2))
            G.paged_read(which, bt, k, v)
            got.append([d.download(np.float32, (rows * (n - 1), n_kv * hd)) for d in (k, v)])
        assert np.array_equal(got[0][0], got[1][0]) and np.array_equal(got[0][1], got[1][1])
    assert kvs[0].status() == 0
