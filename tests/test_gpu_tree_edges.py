"""Draft trees over the paged KV cache where a call can go wrong unseen: pages outside
the pool judged by the right masks."""
import numpy as np
import pytest

from paged_util import F16, Q4_0, Q8_0
from tree_util import TreeCase

pytestmark = pytest.mark.gpu
TYPES = [F16, Q8_0, Q4_0]


def _lose(c, entries):
    """Page ids outside the pool: table entry entries[s] of sequence s."""
    table = c.table.copy()
    table[np.arange(len(c.lens)), entries] = 10 ** 6
    c.d["table"].upload(table)


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
