"""A plain model of draft trees over the paged KV cache, and of beam search's
selection: masks from parents, attention over the positions that a mask leaves,
the greedy walk, and the best candidates in float64."""
import numpy as np

from paged_util import Case, attend


def random_parents(rng, n, roots=0.1):
    """Parents of n tokens: the first has none, the others one of those before, now and then none."""
    return [-1 if i == 0 or rng.random() < roots else int(rng.integers(0, i)) for i in range(n)]


def ancestry(parents):
    """(sets of attended tokens, depths)"""
    sets, depth = [], []
    for i, up in enumerate(parents):
        sets.append((sets[up] if up >= 0 else set()) | {i})
        depth.append(depth[up] + 1 if up >= 0 else 0)
    return sets, depth


def pack(sets, words):
    out = np.zeros((len(sets), words), np.uint32)
    for i, s in enumerate(sets):
        for j in s:
            if j < 32 * words:
                out[i, j // 32] |= np.uint32(1 << (j % 32))
    return out


class TreeCase(Case):
    """A Case whose new tokens form trees: `sets` and `depths`, one per token of the
    batch (random trees unless given), the masks of `words` words."""

    def __init__(self, G, t, n_head, n_kv, hd, page, lens, new, words=None, sets=None, depths=None, seed=0, **more):
        super().__init__(G, t, n_head, n_kv, hd, page, lens, new=new, seed=seed, **more)
        rng = np.random.default_rng(seed + 1)
        self.words = words or max(1, -(-max(self.new + [1]) // 32))
        self.parents = [random_parents(rng, n) for n in self.new]
        trees = [ancestry(p) for p in self.parents]
        self.sets = sets if sets is not None else [s for tree in trees for s in tree[0]]
        self.depths = depths if depths is not None else [d for tree in trees for d in tree[1]]
        mask = np.full((max(1, self.n_tok), self.words), 0xdeadbeef, np.uint32)
        mask[:len(self.sets)] = pack(self.sets, self.words)
        depth = np.full(max(1, self.n_tok), 77, np.int32)
        depth[:len(self.depths)] = self.depths
        B = G.Buffer.from_array
        self.d["mask"], self.d["depth"] = B(mask), B(depth)
        self.tree = G.PagedTree(self.words, self.d["mask"], self.d["depth"])

    def attn(self, scale, cap=0.0, window=0, out=None, **more):
        G = self.G
        out = out or G.Buffer.from_array(np.full((max(1, self.n_tok), self.n_head, self.hd), 7.5, np.float32))
        G.paged_attn_tree(self.kv, self.batch, self.tree, self.d["q"], self.n_head, out, scale=scale, softcap=cap, window=window, **more)
        return out.download(np.float32, (self.n_tok, self.n_head, self.hd))

    def seen(self, s, i, window=0):
        """Indexes into prefix + own rows of what token i of sequence s attends."""
        n, size = self.new[s], self.lens[s]
        first, t = size - n, self.off[s] + i
        if first + i < 0:
            return []
        low = first + min(max(self.depths[t], 0), n - 1) + 1 - window if window else -self.n_prefix
        cached = [self.n_prefix + p for p in range(max(-self.n_prefix, low), max(first, 0))]
        return cached + [self.n_prefix + first + j for j in sorted(self.sets[t]) if j < min(n, 32 * self.words) and first + j >= 0]

    def expect(self, scale, cap=0.0, window=0):
        grp = self.n_head // self.n_kv
        out, tol = np.full((self.n_tok, self.n_head, self.hd), 7.5), np.zeros((self.n_tok, self.n_head, self.hd))
        for s, n in enumerate(self.new):
            for i in range(n):
                t, at = self.off[s] + i, self.seen(s, i, window)
                for h in range(self.n_head):
                    k, v = (np.concatenate([self.shared[w][:, h // grp], self.rows[s][w][:, h // grp]])[at] for w in (0, 1))
                    out[t, h], tol[t, h] = attend(self.q[t, h], k, v, len(at) - 1, scale, cap)
        return out, tol


def walk(parents, tokens, choice, most):
    """(kept tokens, the choice at the last)"""
    if not parents:
        return [], -1
    path = [0]
    while len(path) < most:
        more = [j for j in range(len(parents)) if parents[j] == path[-1] and tokens[j] == choice[path[-1]]]
        if not more:
            break
        path.append(more[0])
    return path, choice[path[-1]]


def select(x, score, n_beam, n_out, ended=None):
    """Beam selection in float64: scores, rows, tokens [group][n_out]."""
    rows, vocab = x.shape
    out = np.full((rows // n_beam, n_out), -np.inf), *(np.full((rows // n_beam, n_out), -1, np.int32) for _ in range(2))
    for g in range(rows // n_beam):
        found = []
        for r in range(g * n_beam, (g + 1) * n_beam):
            s, y = float(score[r]), x[r].astype(np.float64)
            if ended is not None and ended[r]:
                found.append((s, r, np.inf, -1))
                continue
            if np.isnan(y).any() or (y == np.inf).any() or (y == -np.inf).all():
                continue
            top = y.max()
            norm = top + np.log(np.exp(y - top).sum())
            order = np.lexsort((np.arange(vocab), -y))[:n_out]
            found += [(s + (y[v] - norm), r, y[v], int(v)) for v in order]
        found = [f for f in found if f[0] > -np.inf]         # nor a NaN
        found.sort(key=lambda f: (-f[0], f[1], -f[2], f[3]))
        for i, (s, r, _, v) in enumerate(found[:n_out]):
            out[0][g, i], out[1][g, i], out[2][g, i] = s, r, v
    return out
