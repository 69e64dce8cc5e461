"""Draft trees over the paged KV cache where a call can go wrong unseen: pages outside
the pool judged by the right masks, caps far above the scores, windows that a draft outgrows."""
import numpy as np
import pytest

from paged_util import F16, Q4_0, Q8_0, attend
from tree_util import TreeCase, pack

pytestmark = pytest.mark.gpu
TYPES = [F16, Q8_0, Q4_0]


def _lose(c, entries):
    """Page ids outside the pool: table entry entries[s] of sequence s."""
    table = c.table.copy()
    table[np.arange(len(c.lens)), entries] = 10 ** 6
    c.d["table"].upload(table)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("n,first,window", [(6, 29, 2), (6, 20, 0), (6, 16, 0), (7, 16, 3), (20, 18, 4), (20, 16, 0), (40, 27, 6), (40, 33, 30)])
def test_a_bad_page_that_a_row_does_not_attend(gpu, t, hd, n, first, window):
    """Windows that leave a row no cached position, and bits of tokens that the sequence
    does not have: neither makes a row attend the page beside the positions it sees."""
    rng = np.random.default_rng(n + first)
    words = -(-n // 32)
    sets = [{j for j in range(n) if rng.random() < 0.15} | {j for j in range(n, 32 * words) if rng.random() < 0.5} for _ in range(n)]
    depths = [int(rng.integers(0, min(n, 14))) for _ in range(n)]
    c = TreeCase(gpu, t, 2, 1, hd, 16, [first + n], [n], words=words, sets=sets, depths=depths, seed=44)
    clean = c.attn(hd ** -0.5, window=window)
    assert np.isfinite(clean).all() and c.kv.status() == 0
    kept = 0
    for page in range(-(-(first + n) // 16)):
        _lose(c, [page])
        got = c.attn(hd ** -0.5, window=window)
        lost = np.array([any(p // 16 == page for p in c.seen(0, i, window)) for i in range(n)])
        assert np.isnan(got[lost]).all()
        assert np.array_equal(got[~lost], clean[~lost]), (page, np.argwhere(~np.isclose(got, clean).all((1, 2)) & ~lost).ravel())
        assert c.kv.status() == (gpu.PAGED_BAD_PAGE if lost.any() else 0)
        kept += (~lost).sum()
    # (without a window all rows attend every page that holds a cached position)
    assert kept or (window == 0 and (first + n - 1) // 16 == (first - 1) // 16)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd,n_head,n_kv,n", [(64, 4, 2, 20), (128, 4, 2, 20), (256, 65, 1, 3), (512, 2, 1, 20)])
def test_bad_pages_of_drafts_with_unlike_masks(gpu, t, hd, n_head, n_kv, n):
    """A workgroup goes through several drafts, each with a lost page among its first and
    masks of its own: what the one before attended decides nothing."""
    drafts = 330 if n > 3 else 130
    last = {j for j in range(n) if (16 + j) // 16 == (16 + n - 1) // 16}                # the tokens of the lost page
    rng = np.random.default_rng(hd)
    sets = []
    for s in range(drafts):
        for i in range(n):
            some = {j for j in range(n) if rng.random() < 0.5}
            sets.append((some | {max(last)}) if (i + s) % 2 else (some - last))
    c = TreeCase(gpu, t, n_head, n_kv, hd, 16, [16 + n] * drafts, [n] * drafts, sets=sets, seed=40)
    clean = c.attn(hd ** -0.5)
    assert np.isfinite(clean).all() and c.kv.status() == 0
    _lose(c, [(16 + n - 1) // 16] * drafts)
    lost = np.array([bool(x & last) for x in sets])
    for _ in range(3):
        got = c.attn(hd ** -0.5)
        assert np.isnan(got[lost]).all()
        assert np.array_equal(got[~lost], clean[~lost])
        assert c.kv.status() == gpu.PAGED_BAD_PAGE


def _capped(c, scale, cap):
    """Outputs and tolerances as TreeCase.expect's, but with the cap's part relative to
    the capped score, which is small where the cap is large.  tanh to 2^-20 of itself:
    below 0.3 an odd polynomial leaves 9e-3 x^11 out, less than 2^-24 x there, and rounds
    a few times; above it is (1 - t) / (1 + t) with t = exp(-2 x), whose numerator, 0.45
    at least, is off by 2.2 steps of 2^-24 (exponent 0.6, exponential 1.1, difference
    0.5), the rest by 4.4.  The argument's and the result's factors are two roundings more."""
    grp = c.n_head // c.n_kv
    out, tol = np.zeros((c.n_tok, c.n_head, c.hd)), np.zeros((c.n_tok, c.n_head, c.hd))
    for s, n in enumerate(c.new):
        for i in range(n):
            t, at = c.off[s] + i, c.seen(s, i)
            for h in range(c.n_head):
                k, v = (c.rows[s][w][:, h // grp][at] for w in (0, 1))
                q = c.q[t, h].astype(np.float64)
                x = cap * np.tanh(k @ q * scale / cap)
                size = (np.abs(k) @ np.abs(q) * scale).max()
                d = size * (2.0 ** -21 + c.hd * 2.0 ** -24) + np.abs(x).max() * (2.0 ** -20 + 2.0 ** -22) + 2.0 ** -22
                w = np.exp(x - x.max())
                out[t, h] = w @ v / w.sum()
                tol[t, h] = (2 * d + 2.0 ** -18) * (w @ np.abs(v)) / w.sum() + 2.0 ** -29 * len(v) * np.abs(v).max() / w.sum()
    return out, tol


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("new", [[3, 1], [20, 7]])
@pytest.mark.parametrize("cap", [2.0 ** -100, 1e-3, 1.0, 50.0, 1e3, 1e4, 1e6, 1e8, 2.0 ** 100])
def test_caps_of_any_size(gpu, t, hd, new, cap):
    scale = hd ** -0.5
    c = TreeCase(gpu, t, 4, 2, hd, 16, [n + 40 for n in new], new, sets=[set(range(i + 1)) for n in new for i in range(n)],
                 depths=[i for n in new for i in range(n)], spread=1.5, seed=41)
    want, tol = _capped(c, scale, cap)
    got = c.attn(scale, cap=cap)
    assert (np.abs(got - want) <= tol).all(), np.nanmax(np.abs(got - want) / tol)
    # chains: as rows of tokens
    same = gpu.Buffer(got.nbytes)
    gpu.paged_attn(c.kv, c.batch, c.d["q"], 4, same, scale=scale, softcap=cap)
    same = same.download(np.float32, got.shape)
    assert (np.abs(same - want) <= tol).all(), np.nanmax(np.abs(same - want) / tol)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd,n_head", [(256, 65), (512, 33)])
@pytest.mark.parametrize("cap", [1e5, 2.0 ** 100])
def test_large_caps_of_many_query_heads(gpu, t, hd, n_head, cap):
    c = TreeCase(gpu, t, n_head, 1, hd, 16, [40, 22], [2, 3], spread=1.5, seed=42)
    want, tol = _capped(c, hd ** -0.5, cap)
    got = c.attn(hd ** -0.5, cap=cap)
    assert (np.abs(got - want) <= tol).all(), np.nanmax(np.abs(got - want) / tol)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("new", [[3, 1], [20, 7]])
@pytest.mark.parametrize("cap", [20.0, 300.0, 1e3, 1e4])
def test_caps_of_scores_of_one_product(gpu, t, hd, new, cap):
    """A query of one element: the score is one product of two halves, or of a quant and
    its scale, and what is left to be wrong is the cap."""
    c = TreeCase(gpu, t, 4, 2, hd, 16, [n + 40 for n in new], new, seed=43)
    c.q[:] = 0.0
    c.q[:, :, 37] = 1.0
    c.d["q"].upload(c.q)
    got = c.attn(1.0, cap=cap)
    for s, n in enumerate(c.new):
        for i in range(n):
            at = c.seen(s, i)
            for h in range(4):
                k, v = (c.rows[s][w][:, h // 2][at] for w in (0, 1))
                x = cap * np.tanh(k[:, 37] / cap)
                w = np.exp(x - x.max())
                # the product and its factors 2^-22 (four roundings), tanh 2^-20, the exponential 2^-22
                d = np.abs(x).max() * (2.0 ** -20 + 2.0 ** -21) + 2.0 ** -22
                tol = (2 * d + 2.0 ** -18) * (w @ np.abs(v)) / w.sum() + 2.0 ** -29 * len(v) * np.abs(v).max() / w.sum()
                off = np.abs(got[c.off[s] + i, h] - w @ v / w.sum())
                assert (off <= tol).all(), (s, i, h, (off / tol).max())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("new,window", [([6], 3), ([6, 2], 6), ([40, 9], 8), ([40], 33), ([40], 39), ([40], 40)])
@pytest.mark.parametrize("chain", [True, False])
def test_a_window_that_a_draft_outgrows(gpu, t, new, window, chain):
    """Masks without the ancestors that a token's window has left: its attention is that of
    the row of tokens that it continues, with this window."""
    c = TreeCase(gpu, t, 4, 2, 128, 16, [n + 50 for n in new], new, n_prefix=11, seed=45)
    parents = [list(range(-1, n - 1)) if chain else [-1] + [max(0, i - 1 - (i * 7) % 3) for i in range(1, n)] for n in new]
    paths, at = [], 0
    for up in parents:
        for i, x in enumerate(up):
            paths.append((paths[at + x] if x >= 0 else []) + [i])
        at += len(up)
    c.sets, c.depths = [set(p[-window:]) for p in paths], [len(p) - 1 for p in paths]
    assert max(c.depths) + 1 >= min(window, 3)
    c.d["mask"].upload(pack(c.sets, c.words))
    c.d["depth"].upload(np.asarray(c.depths, np.int32))
    got = c.attn(0.1, window=window)
    for s, n in enumerate(c.new):
        first = c.n_prefix + c.lens[s] - n
        for i in range(n):
            tok = c.off[s] + i
            row = list(range(first)) + [first + j for j in paths[tok]]
            for h in range(4):
                k, v = (np.concatenate([c.shared[w][:, h // 2], c.rows[s][w][:, h // 2]])[row] for w in (0, 1))
                want, tol = attend(c.q[tok, h], k, v, len(row) - 1, 0.1, window=window)
                assert (np.abs(got[tok, h] - want) <= tol).all(), (s, i, h)
    if chain:
        same = gpu.Buffer(got.nbytes)
        gpu.paged_attn(c.kv, c.batch, c.d["q"], 4, same, scale=0.1, window=window)
        want, tol = super(TreeCase, c).expect(0.1, window=window)
        assert (np.abs(same.download(np.float32, got.shape) - got) <= 2 * tol).all()
