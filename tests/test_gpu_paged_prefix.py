"""Attention over the paged KV cache behind a short shared prefix, with more steps
than workgroups: a workgroup's share then holds several whole tiles of the prefix."""
import numpy as np
import pytest

from paged_util import F16, Q4_0, Q8_0, Case, LongCase

pytestmark = pytest.mark.gpu
TYPES = [F16, Q8_0, Q4_0]
IDS = ["f16", "q8_0", "q4_0"]


@pytest.mark.parametrize("n_prefix,window,cap", [(0, 0, 0.0), (40, 0, 20.0), (40, 25, 0.0)])
@pytest.mark.parametrize("t", TYPES, ids=IDS)
def test_long_case_is_a_case(gpu, t, n_prefix, window, cap):
    # the array-wise twin of the plain model gives the same batch and the same answers
    a, b = (kind(gpu, t, 4, 2, 64, 16, [30, 7, 0], new=[9, 7, 2], pad=1, n_prefix=n_prefix, seed=50) for kind in (Case, LongCase))
    b.q[:] = a.q
    for s in range(4):
        src, dst = (x.shared if s == 3 else x.rows[s] for x in (a, b))
        pages = a.prefix if s == 3 else a.table[s]
        for w in (0, 1):
            for p in range(len(dst[w])):
                for h in range(2):
                    assert np.array_equal(b.pool.get(bool(w), pages[p // 16], p % 16, h), dst[w][p, h])
            dst[w][:] = src[w]
    want, got = a.expect(0.2, cap, window), b.expect(0.2, cap, window)
    assert np.allclose(want[0], got[0], rtol=1e-12, atol=1e-12)
    assert np.all(got[1] >= want[1] * (1 - 1e-9))


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("hd,n_head,n_kv,lens,new,n_prefix", [
    (64, 8, 8, [8192, 8190, 8000, 8100], None, 100),
    (128, 8, 8, [8192, 7000, 8000], None, 40),
    (128, 16, 8, [4000, 3990, 4010, 3000], [2, 1, 1, 1], 90),
    (256, 8, 8, [4000, 3900, 4090], None, 60),
    (512, 8, 8, [2000, 2500], None, 30),
])
def test_long_conversations_behind_a_short_prefix(gpu, t, hd, n_head, n_kv, lens, new, n_prefix):
    LongCase(gpu, t, n_head, n_kv, hd, 64, lens, new=new, n_prefix=n_prefix, seed=hd + n_head).check()


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("hd,n_head,n_kv", [(64, 32, 8), (128, 32, 8), (256, 16, 4), (512, 8, 4)])
@pytest.mark.parametrize("window", [0, 70])
def test_prompts_behind_a_short_prefix(gpu, t, hd, n_head, n_kv, window):
    LongCase(gpu, t, n_head, n_kv, hd, 16, [256, 300, 200, 256], new=[256, 211, 200, 1], pad=2, n_prefix=50, seed=hd).check(window=window)


@pytest.mark.parametrize("t", TYPES, ids=IDS)
def test_prompts_behind_a_prefix_of_hundreds(gpu, t):
    # shares of a part of a prefix tile, whole ones, and own tiles
    LongCase(gpu, t, 16, 4, 128, 32, [200] * 6, new=[200, 150, 3, 1, 200, 90], n_prefix=333, seed=51).check(cap=30.0)


@pytest.mark.parametrize("t", TYPES, ids=IDS)
def test_graph_replays_with_other_shares(gpu, t):
    """A captured call whose shares hold whole tiles of the prefix, or parts, as the
    lengths change; eager calls over a workspace of their own between the replays."""
    G = gpu
    full = [8000, 7000, 6500, 5]
    c = LongCase(G, t, 16, 8, 128, 64, full, n_prefix=40, seed=52)
    s, rows = G.Stream(), [x[:] for x in c.rows]
    ws = G.Buffer.from_array(np.full(G.paged_attn_workspace_bytes(c.kv, c.batch, 16), 0xff, np.uint8))
    out = G.Buffer.from_array(np.full((4, 16, 128), 7.5, np.float32))
    g = G.Graph(s.ptr, lambda: G.paged_attn(c.kv, c.batch, c.d["q"], 16, out, scale=0.1, ws=ws, stream=s.ptr))
    for step, lens in enumerate([full, [60, 5, 0, 1], [8000, 1, 6000, 5], full]):
        c.lens = lens
        c.rows = [[w[:n] for w in x] for x, n in zip(rows, lens)]
        c.d["lens"].upload(np.asarray(lens + [0], np.int32), s.ptr)
        g.launch(s.ptr)
        s.synchronize()
        got = out.download(np.float32, (4, 16, 128))
        want, tol = c.expect(0.1)
        assert np.all(np.abs(got - want) <= tol), step
        assert np.array_equal(c.attn(0.1), got), step
    assert c.kv.status() == 0
