"""Several continuations of a sequence over a paged key/value cache, as runnable cases.

Drafted tokens that form a tree are appended and attended in one call, each seeing
the cached positions and its own ancestors; the greedy walk accepts a path, whose
rows are moved together in the caches of all layers.  Beam search selects the best
continuations over beams and vocabulary, and the surviving beams' page tables and
part-filled pages are laid out anew.  `listed()` names the cases, `draw()` makes
others of the same ranges, `prepare()` makes a case's inputs on the GPU, and `run()`
is one pass: in elementary torch operations, or, with `own` set, through the public
entry points of g4run_amd.  `exact()` computes the same values in 64 bits.

Page layout of the pools (page slots a multiple of 16):
  f16         [n_kv][slot][hd] halves
  q8_0, q4_0  the quants of [n_kv][slot] rows, then the rows' fp16 scales
              [n_kv][slot][hd / 32].  With e = 32 s + 8 g + j (key rows) and
              e = 16 m + c (value rows):
              q8_0 keys: byte g hd/4 + 8 s + j, values: byte c hd/16 + m, each
              holding quant + 128;
              q4_0 keys: nibble (j >> 1) + 4 (j & 1) of the dword g hd/32 + s,
              values: nibble m of the hd/16 that start at byte c hd/32.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"f16": 1, "q4_0": 2, "q8_0": 8}
LARGEST = 16 * 8192 * 8 * 128              # key elements of the largest batch
MOST = 32 * 64 * 32768 * 128               # (head, token, key) products of the largest batch, by element
LOGITS = 16 * 8 * 262144                   # of the largest selection
POOLS = 52 * 80 * 64 * 4 * 256             # elements of the largest caches whose rows are moved


def listed():
    gemma = dict(n_head=8, n_kv=4, hd=256)     # the synthetic decoder's heads
    wide = dict(n_head=32, n_kv=8, hd=128)
    layers = dict(n_cache=26, n_kv=4, hd=256)  # the caches of the synthetic decoder's layers
    return [
        # one conversation's draft of 8 tokens over a short cache, the whole step of a layer: latency
        _tree("tree_step_f16", "f16", n_seq=1, max_len=100, new=8, step=True, **gemma),
        # a wide draft of 64 tokens at the end of one long document
        _tree("tree_long_f16", "f16", n_seq=1, max_len=32768, new=64, page=64, **wide),
        # 16 conversations of up to 8192 positions, drafts of up to 16 tokens each: bandwidth
        _tree("tree_batch_f16", "f16", n_seq=16, max_len=8192, new=16, page=64, **wide),
        # 32 conversations over 8-bit pages, drafts of up to 33 tokens, capped scores
        _tree("tree_batch_q8_0_cap", "q8_0", n_seq=32, max_len=4096, new=33, cap=50.0, **gemma),
        # sliding-window layers of wide heads over 4-bit pages, behind a prefix that all share
        _tree("tree_window_q4_0", "q4_0", n_seq=8, max_len=3000, new=24, window=1024, page=16, n_prefix=500, n_head=8, n_kv=2, hd=512),
        # the accepted path of one conversation's draft, all layers: latency
        _keep("keep_one_f16", "f16", n_seq=1, max_len=200, new=16, most=5, **layers),
        # the accepted paths of 32 drafts of 64 tokens, 8-bit caches of all layers
        _keep("keep_batch_q8_0", "q8_0", n_seq=32, max_len=300, new=64, most=9, n_cache=26, n_kv=8, hd=128),
        # one request's 4 beams over a small vocabulary: latency
        _beam("beam_one", n_group=1, n_beam=4, n_vocab=32768, n_out=8),
        # 64 requests of 4 beams, rows of odd length
        _beam("beam_odd", n_group=64, n_beam=4, n_vocab=50001, n_out=4),
        # 16 requests of 8 beams over the largest vocabulary: bandwidth
        _beam("beam_batch", n_group=16, n_beam=8, n_vocab=262144, n_out=16),
        # one request's beams carried over, all layers: latency
        _fork("fork_one_f16", "f16", n_group=1, n_beam=4, max_len=90, page=32, **layers),
        # 4 requests' beams, pages of 64 positions, all layers: bandwidth
        _fork("fork_batch_f16", "f16", n_group=4, n_beam=8, max_len=300, page=64, **layers),
    ]


def _named(name, base, more):
    return ({"name": name} if name else {}) | base | more


def _tree(name, kv, **more):
    return _named(name, dict(kind="tree", kv=kv, page=32, step=False, n_prefix=0, cap=0.0, window=0), more)


def _keep(name, kv, **more):
    return _named(name, dict(kind="keep", kv=kv, page=32), more)


def _beam(name, **more):
    return _named(name, dict(kind="beam"), more)


def _fork(name, kv, **more):
    return _named(name, dict(kind="fork", kv=kv), more)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "tree", "keep", "beam", "beam", "fork"])
    if kind == "beam":
        n_beam = rng.choice([1, 2, 3, 4, 5, 8, 16, 32])
        n_out = rng.choice([n_beam, min(64, 2 * n_beam)])
        n_vocab = _log(rng, 1000, 262144)
        return _beam(None, n_group=_log(rng, 1, min(64, LOGITS // (n_beam * n_vocab))), n_beam=n_beam, n_vocab=n_vocab, n_out=n_out)
    kv, page = rng.choice(["f16", "f16", "q8_0", "q4_0"]), rng.choice([16, 32, 48, 64, 128])
    hd = rng.choice([64, 128, 128, 256, 256, 512])
    n_kv = rng.choice([1, 2, 4, 8] if hd < 512 else [1, 2])
    if kind == "keep":
        n_cache, new = _log(rng, 1, 32), _log(rng, 2, 100)
        n_seq = _log(rng, 1, max(1, min(32, POOLS // (2 * n_cache * n_kv * hd * (new + 260)))))
        return _keep(None, kv, n_seq=n_seq, max_len=new + _log(rng, 1, 200), new=new, most=_log(rng, 1, 12), n_cache=n_cache, n_kv=n_kv, hd=hd, page=page)
    if kind == "fork":
        n_cache, n_beam, max_len = _log(rng, 1, 32), rng.choice([2, 3, 4, 5, 8]), _log(rng, 1, 300)
        pages = max_len // page + 3 * n_beam
        n_group = _log(rng, 1, max(1, min(16, POOLS // (2 * n_cache * n_kv * hd * page * pages))))
        return _fork(None, kv, n_group=n_group, n_beam=n_beam, max_len=max_len, page=page, n_cache=n_cache, n_kv=n_kv, hd=hd)
    n_head = n_kv * rng.choice([1, 2, 3, 4, 8] if hd < 512 else [1, 2, 4])
    n_prefix = rng.choice([0, 0, 0, _log(rng, 20, 2000)])
    new = _log(rng, 1, 160)
    n_seq = _log(rng, 1, max(1, min(48, MOST // (n_head * hd * new * (new + n_prefix + 200)))))
    most = min(LARGEST // (n_seq * n_kv * hd), MOST // (n_seq * new * n_head * hd) - n_prefix)
    return _tree(None, kv, n_seq=n_seq, max_len=new + _log(rng, 1, max(2, min(16384, most - new))), new=new, step=kv == "f16" and rng.random() < 0.3,
                 n_prefix=n_prefix, cap=rng.choice([0.0, 0.0, 30.0]), window=rng.choice([0, 0, 512]), n_head=n_head, n_kv=n_kv, hd=hd, page=page)


# ------------------------------------------------------------------- the inputs
def _frac(i):
    return (0.5 + 0.6180339887498949 * i) % 1.0


def _new(c):
    """New tokens of each sequence: the first has the most."""
    return [c["new"] if i == 0 else 1 + int((c["new"] - 1) * _frac(i)) for i in range(c["n_seq"])]


def _lens(c):
    """Positions in each sequence's own pages, its new tokens included."""
    return [c["max_len"] if i == 0 else n + int((c["max_len"] - n) * _frac(i + 7)) for i, n in enumerate(_new(c))]


def _kept(c):
    """Accepted tokens of each sequence."""
    return [min((n + 1) // 2, c["most"] if i == 0 else 1 + int((c["most"] - 1) * _frac(i + 3))) for i, n in enumerate(_new(c))]


def _sizes(c):
    """Positions of each beam, those of one request alike."""
    return [c["max_len"] if g == 0 else 1 + int((c["max_len"] - 1) * _frac(g)) for g in range(c["n_group"]) for _ in range(c["n_beam"])]


def _row(c):
    """Bytes of one cached row."""
    return c["hd"] * 2 if c["kv"] == "f16" else c["hd"] // (1 if c["kv"] == "q8_0" else 2) + c["hd"] // 16


def _pool(c, gen, *lead):
    """Pages [*lead, page's data] whose rows hold values of unit size."""
    h, p, d = c["n_kv"], c["page"], c["hd"]
    if c["kv"] == "f16":
        return torch.randn(*lead, h, p, d, device="cuda", generator=gen, dtype=torch.float16)
    sc = torch.rand(*lead, h * p * (d // 32), device="cuda", generator=gen) * 0.5 + 0.75
    if c["kv"] == "q8_0":
        q = torch.randn(*lead, h * p * d, device="cuda", generator=gen, dtype=torch.float16) * 42
        q, sc = q.clamp_(-127, 127).round_().add_(128).to(torch.uint8), (sc / 42).half()
    else:
        q = torch.randn(2, *lead, h * p * d // 2, device="cuda", generator=gen, dtype=torch.float16) * 2.6
        q = q.clamp_(-8, 7).round_().add_(8).to(torch.uint8)
        q = q[0] | (q[1] << 4)
        sc = (sc / -2.6).half()
    return torch.cat([q, sc.view(torch.uint8)], -1)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    if c["kind"] == "beam":
        rows = c["n_group"] * c["n_beam"]
        x = rand(rows, c["n_vocab"]).mul_(2.5).add_(rand(rows, 1) * 3)
        banned = torch.randint(c["n_vocab"], (rows, 5), device="cuda", generator=gen)
        x.scatter_(1, banned, -math.inf)
        score = -torch.rand(rows, device="cuda", generator=gen) * 4
        ended = (torch.rand(rows, device="cuda", generator=gen) < 0.1).int()
        beam, group = torch.arange(rows, device="cuda") % c["n_beam"], torch.arange(rows, device="cuda") // c["n_beam"]
        first = group % 5 == 4                               # a request's first step: its first beam alone
        score = torch.where(first & (beam > 0), -math.inf, score)
        return dict(c=c, x=x, score=score, ended=torch.where(first, 0, ended).int(), kept={})
    if c["kind"] == "fork":
        rows, sizes, p = c["n_group"] * c["n_beam"], _sizes(c), c["page"]
        width = c["max_len"] // p + 1
        table, at = torch.full((rows, width), -1, dtype=torch.int32), 0
        whole = [n // p for n in sizes[::c["n_beam"]]]
        order = torch.randperm(sum(whole) + 2 * rows + 3, generator=host).to(torch.int32)
        for g, n in enumerate(whole):                        # whole pages shared by a request's beams
            table[g * c["n_beam"]:(g + 1) * c["n_beam"], :n] = order[at:at + n]
            at += n
        for i, n in enumerate(sizes):
            if n % p:
                table[i, n // p] = order[at + i]
        parent = torch.randint(c["n_beam"], (rows,), generator=host) + torch.arange(rows) // c["n_beam"] * c["n_beam"]
        return dict(c=c, lens=_ints(sizes), table=table.cuda(), parent=parent.int().cuda(), fresh=order[at + rows:at + 2 * rows].cuda(),
                    len_out=_ints([0] * rows), table_out=torch.full((rows, width), -1, dtype=torch.int32).cuda(),
                    k_pool=_pool(c, gen, c["n_cache"], len(order)), v_pool=_pool(c, gen, c["n_cache"], len(order)), kept={})
    new, lens = _new(c), _lens(c)
    n_tok = sum(new)
    pages = [-(-n // c["page"]) for n in lens]
    n_pre = -(-c.get("n_prefix", 0) // c["page"])
    order = torch.randperm(sum(pages) + n_pre + 3, generator=host).to(torch.int32)
    table, at = torch.full((c["n_seq"], max(pages)), -1, dtype=torch.int32), 0
    for i, n in enumerate(pages):
        table[i, :n] = order[at:at + n]
        at += n
    st = dict(c=c, n_tok=n_tok, lens=_ints(lens), table=table.cuda(), q_off=_ints([sum(new[:i]) for i in range(len(new) + 1)]), kept={})
    u = torch.rand(n_tok, generator=host).tolist()
    if c["kind"] == "keep":
        # the accepted path: token 0, then some behind the places that the path's rows move to
        vocab, parent, token = 262144, [], []
        choice = torch.randint(vocab, (n_tok,), generator=host).tolist()
        t = 0
        for n, k in zip(new, _kept(c)):
            path = [0] + sorted((k + torch.randperm(n - k, generator=host)[:k - 1]).tolist())
            up = dict(zip(path[1:], path))
            par = [-1] + [up.get(i, max(0, i - 8) + int(u[t + i] * min(i, 8))) for i in range(1, n)]
            parent += par
            token += [(choice[t + max(0, par[i])] + (0 if i in up else 1)) % vocab for i in range(n)]
            t += n
        pool = c["n_cache"], len(order)
        return st | dict(parent=_ints(parent), token=_ints(token), choice=_ints(choice), n_keep=_ints([0] * c["n_seq"]), next=_ints([0] * c["n_seq"]),
                         len_out=_ints([0] * c["n_seq"]), keep=_ints([[0] * c["most"]] * c["n_seq"]), k_pool=_pool(c, gen, *pool), v_pool=_pool(c, gen, *pool))
    words = -(-max(new) // 32)
    parent, mask, depth, t = [], [], [], 0
    for n in new:
        m, d = [], []
        for i in range(n):
            up = max(0, i - 8) + int(u[t + i] * min(i, 8)) if i else -1
            m.append((m[up] if i else 0) | 1 << i)
            d.append(d[up] + 1 if i else 0)
            parent.append(up)
        mask += [[(x >> 32 * w) & 0xffffffff for w in range(words)] for x in m]
        depth += d
        t += n
    mask = torch.tensor(mask, dtype=torch.int64)
    st |= dict(words=words, parent=_ints(parent), mask=torch.where(mask >= 2 ** 31, mask - 2 ** 32, mask).int().cuda(), depth=_ints(depth),
               prefix=order[at:at + n_pre].cuda(), k_pool=_pool(c, gen, len(order)), v_pool=_pool(c, gen, len(order)),
               q=rand(n_tok, c["n_head"], c["hd"]) * 1.5, out=torch.zeros(n_tok, c["n_head"], c["hd"], device="cuda"))
    if c["step"]:
        st |= dict(q_out=torch.zeros_like(st["q"]), k=rand(n_tok, c["n_kv"], c["hd"]), v=rand(n_tok, c["n_kv"], c["hd"]),
                   mask=torch.zeros_like(st["mask"]), depth=torch.zeros_like(st["depth"]))
    return st


def run(state):
    kind = state["c"]["kind"]
    if own:
        return {"tree": _own_tree, "keep": _own_keep, "beam": _own_beam, "fork": _own_fork}[kind](state)
    return {"tree": _plain_tree, "keep": _plain_keep, "beam": _plain_beam, "fork": _plain_fork}[kind](state)


# ---------------------------------------------- the library's own entry points
def _plan(st):
    """The caches, the batch's description and the workspace, which a serving
    loop keeps from call to call."""
    if not st["kept"]:
        import g4run_amd as G
        G.init()
        c, p = st["c"], dict(G=G)
        if c["kind"] == "beam":
            p["ws"] = G.Buffer(max(16, G.beam_workspace_bytes(c["n_group"], c["n_beam"], c["n_vocab"], c["n_out"])))
        else:
            pools = [(st["k_pool"], st["v_pool"])] if c["kind"] == "tree" else list(zip(st["k_pool"], st["v_pool"]))
            p["kv"] = [G.PagedKV(TYPES[c["kv"]], c["n_kv"], c["hd"], c["page"], k.shape[0], k=k.data_ptr(), v=v.data_ptr()) for k, v in pools]
            p["batch"] = G.PagedBatch(len(st["lens"]), st.get("n_tok", 0), st["lens"].data_ptr(), st["table"].data_ptr(), st["table"].shape[1], c["max_len"],
                                      q_off=st["q_off"].data_ptr() if "q_off" in st else None, n_prefix=c.get("n_prefix", 0),
                                      prefix=st["prefix"].data_ptr() if c.get("n_prefix") else None)
        if c["kind"] in ("keep", "fork"):
            p["caches"] = G.PagedCaches(p["kv"])
        if c["kind"] == "tree":
            p["tree"] = G.PagedTree(st["words"], st["mask"].data_ptr(), st["depth"].data_ptr())
            p["rope"] = G.Rope(c["hd"], 1e6)
            p["ws"] = G.Buffer(max(16, G.paged_attn_tree_workspace_bytes(p["kv"][0], p["batch"], c["n_head"])))
        st["kept"] = p
    return st["kept"]


def _own_tree(st):
    p, c, G = _plan(st), st["c"], _plan(st)["G"]
    q = st["q"]
    if c["step"]:
        q = st["q_out"]
        G.paged_tree_build(p["batch"], st["parent"].data_ptr(), st["words"], st["mask"].data_ptr(), st["depth"].data_ptr())
        G.paged_append_tree(p["kv"][0], p["batch"], p["tree"], st["k"].data_ptr(), st["v"].data_ptr(), q=st["q"].data_ptr(), q_out=q.data_ptr(),
                            n_head=c["n_head"], rope=p["rope"])
    G.paged_attn_tree(p["kv"][0], p["batch"], p["tree"], q.data_ptr(), c["n_head"], st["out"].data_ptr(), scale=c["hd"] ** -0.5, softcap=c["cap"],
                      window=c["window"], ws=p["ws"])
    if c["step"]:
        return {"out": st["out"], "mask": st["mask"], "depth": st["depth"], "k": st["k_pool"], "v": st["v_pool"]}
    return {"out": st["out"]}


def _own_keep(st):
    p, c, G = _plan(st), st["c"], _plan(st)["G"]
    G.paged_tree_accept(p["batch"], st["parent"].data_ptr(), st["token"].data_ptr(), st["choice"].data_ptr(), c["most"], st["n_keep"].data_ptr(),
                        st["keep"].data_ptr(), next_out=st["next"].data_ptr(), len_out=st["len_out"].data_ptr())
    G.paged_keep(p["caches"], p["batch"], st["n_keep"].data_ptr(), st["keep"].data_ptr(), c["most"])
    return {n: st[n] for n in ("n_keep", "keep", "next", "len_out", "k_pool", "v_pool")}


def _own_beam(st):
    p, c, G = _plan(st), st["c"], _plan(st)["G"]
    n = c["n_group"], c["n_out"]
    score = torch.empty(n, device="cuda")
    row, token = (torch.empty(n, device="cuda", dtype=torch.int32) for _ in range(2))
    G.beam_select(st["x"].data_ptr(), c["n_group"], c["n_beam"], c["n_vocab"], st["score"].data_ptr(), c["n_out"], score.data_ptr(), row.data_ptr(),
                  token.data_ptr(), ended=st["ended"].data_ptr(), ws=p["ws"])
    return {"score": score, "row": row, "token": token}


def _own_fork(st):
    p = _plan(st)
    p["G"].paged_fork(p["caches"], p["batch"], len(st["parent"]), st["parent"].data_ptr(), st["fresh"].data_ptr(), st["len_out"].data_ptr(),
                      st["table_out"].data_ptr(), st["table_out"].shape[1])
    return {n: st[n] for n in ("len_out", "table_out", "k_pool", "v_pool")}


# ------------------------------------------------------------- the plain forms
def _values(c, raw, value):
    """Pages ([..., page's data]) as 32-bit values [..., n_kv, slot, hd]."""
    if c["kv"] == "f16":
        return raw.float()
    h, p, d = c["n_kv"], c["page"], c["hd"]
    lead = raw.shape[:-1]
    n = h * p * d // (1 if c["kv"] == "q8_0" else 2)
    b = raw[..., :n].reshape(*lead, h, p, -1)
    sc = raw[..., n:].contiguous().view(torch.float16).float().reshape(*lead, h, p, d // 32, 1)
    if c["kv"] == "q8_0":
        q = b.reshape(*lead, h, p, *((16, d // 16) if value else (4, d // 32, 8))).float() - 128
        q = q.transpose(-1, -2) if value else q.transpose(-2, -3)
    elif value:
        b = b.reshape(*lead, h, p, 16, d // 32)
        q = torch.stack([b & 15, b >> 4], -1).flatten(-2).transpose(-1, -2).float() - 8
    else:
        b = b.reshape(*lead, h, p, 4, d // 32, 4)            # nibble pairs (0, 1), (2, 3), ... of a dword: j = 0 2 4 6 1 3 5 7
        q = torch.stack([b & 15, b >> 4], -1).reshape(*lead, h, p, 4, d // 32, 2, 4).transpose(-1, -2).flatten(-2).transpose(-2, -3).float() - 8
    return (q.reshape(*lead, h, p, d // 32, 32) * sc).reshape(*lead, h, p, d)


def _dense(c, pool, table, value):
    """The rows of a page table's sequences, [n_seq, n_kv, positions, hd]."""
    return _values(c, pool[table.clamp(min=0).long()], value).transpose(1, 2).flatten(2, 3)


def _sequence(st):
    """Of every new token: its sequence, its number in it and its slot."""
    tok = torch.arange(st["n_tok"], device="cuda")
    seq = torch.searchsorted(st["q_off"][1:].long(), tok, right=True)
    i = tok - st["q_off"][seq]
    return seq, i, i + st["lens"][seq] - st["q_off"].diff()[seq]


def _ancestry(st, seq, i, n):
    """[token, n]: whether new token j of its sequence is an ancestor, or itself."""
    up = torch.zeros(st["c"]["n_seq"], n, n, device="cuda")
    has = st["parent"] >= 0
    up[seq[has], i[has], st["parent"][has].long()] = 1
    up += torch.eye(n, device="cuda")
    for _ in range(max(1, (n - 1).bit_length())):
        up = (up @ up).clamp(max=1)
    return up[seq, i] > 0


def _packed(sees, words):
    """Truth values [token, n] as 32-bit words."""
    b = torch.nn.functional.pad(sees.long(), (0, 32 * words - sees.shape[1])).reshape(-1, words, 32)
    w = (b << torch.arange(32, device="cuda")).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).int()


def _bits(mask, n):
    return ((mask[:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1).flatten(1)[:, :n] > 0


def _plain_tree(st):
    c, hd, grp = st["c"], st["c"]["hd"], st["c"]["n_head"] // st["c"]["n_kv"]
    s, n, pre = c["n_seq"], c["new"], c["n_prefix"]
    seq, i, slot = _sequence(st)
    q, depth = st["q"], st["depth"]
    if c["step"]:
        bits = _ancestry(st, seq, i, n)
        depth = bits.sum(-1).int() - 1
        freq = 1e6 ** (-2 * torch.arange(hd // 2, device="cuda", dtype=torch.float64) / hd)
        ang = (pre + slot - i + depth).double()[:, None, None] * freq
        cos, sin = torch.cos(ang).float(), torch.sin(ang).float()
        turn = lambda x: torch.cat([x[..., :hd // 2] * cos - x[..., hd // 2:] * sin, x[..., hd // 2:] * cos + x[..., :hd // 2] * sin], -1)  # noqa: E731
        page, at = st["table"][seq, slot // c["page"]].long(), slot % c["page"]
        head = torch.arange(c["n_kv"], device="cuda")
        st["k_pool"][page[:, None], head, at[:, None].long()] = turn(st["k"]).half()
        st["v_pool"][page[:, None], head, at[:, None].long()] = st["v"].half()
        q = turn(q)
    else:
        bits = _bits(st["mask"], n)
    # rows in a rectangle [seq, new], tokens that a sequence does not have seeing nothing
    pick = (st["q_off"][:-1, None] + torch.arange(n, device="cuda")).clamp(max=st["n_tok"] - 1).long()
    q = q[pick].reshape(s, n, c["n_kv"], grp, hd).permute(0, 2, 3, 1, 4).reshape(s, c["n_kv"], grp * n, hd)
    k, v = (_dense(c, st[p], st["table"], p == "v_pool") for p in ("k_pool", "v_pool"))
    sc = q @ k.transpose(-1, -2)
    if pre:
        kp, vp = (_dense(c, st[p], st["prefix"][None], p == "v_pool")[0, :, :pre] for p in ("k_pool", "v_pool"))
        qp = q.transpose(0, 1).reshape(c["n_kv"], -1, hd)
        sc = torch.cat([(qp @ kp.transpose(-1, -2)).reshape(c["n_kv"], s, grp * n, pre).transpose(0, 1), sc], -1)
    sc = sc * hd ** -0.5
    if c["cap"]:
        sc = c["cap"] * torch.tanh(sc / c["cap"])
    base = (st["lens"] - st["q_off"].diff())[:, None, None]
    key = torch.arange(-pre, sc.shape[-1] - pre, device="cuda")
    seen = (key < base).expand(s, n, -1)
    if c["window"]:
        seen = seen & (key > base + depth[pick][..., None] - c["window"])
    j = key - base                                           # of the new tokens
    seen = seen | ((j >= 0) & (j < n) & bits[pick].gather(2, j.clamp(0, n - 1).expand(s, n, -1)))
    sc = sc.reshape(s, c["n_kv"], grp, n, -1).masked_fill(~seen[:, None, None], -math.inf).reshape(sc.shape)
    e = torch.exp(sc - sc.amax(-1, keepdim=True).clamp(min=-3e38))
    o = e[..., pre:] @ v
    if pre:
        o += (e[..., :pre].transpose(0, 1).reshape(c["n_kv"], -1, pre) @ vp).reshape(c["n_kv"], s, grp * n, hd).transpose(0, 1)
    o = o / e.sum(-1, keepdim=True).clamp(min=1e-30)
    out = {"out": o.reshape(s, c["n_head"], n, hd)[seq, :, i]}
    if c["step"]:
        out |= {"mask": _packed(bits, st["words"]), "depth": depth, "k": st["k_pool"], "v": st["v_pool"]}
    return out


def _runs(c, pool):
    """A cache's pools as bytes [cache, page, n_kv, slot, bytes]: the rows, and quantized rows' scales."""
    b = pool.view(torch.uint8).reshape(pool.shape[0], pool.shape[1], -1)
    h, p, d = c["n_kv"], c["page"], c["hd"]
    w = _row(c) if c["kv"] == "f16" else _row(c) - d // 16
    rows = b[..., :h * p * w].unflatten(-1, (h, p, w))
    return [rows] if c["kv"] == "f16" else [rows, b[..., h * p * w:].unflatten(-1, (h, p, d // 16))]


def _move(st, from_page, from_slot, to_page, to_slot):
    """Copies rows of all caches, all of them read before one is written."""
    for pool in (st["k_pool"], st["v_pool"]):
        for x in _runs(st["c"], pool):
            x[:, to_page, :, to_slot] = x[:, from_page, :, from_slot]


def _plain_keep(st):
    c = st["c"]
    s, n, most = c["n_seq"], c["new"], c["most"]
    seq, i, slot = _sequence(st)
    shape = s, n
    parent, token, choice = (torch.full(shape, -2, device="cuda", dtype=torch.int32) for _ in range(3))
    parent[seq, i], token[seq, i], choice[seq, i] = st["parent"], st["token"], st["choice"]
    at = torch.zeros(s, device="cuda", dtype=torch.int64)
    keep, alive, last = [at], torch.ones(s, device="cuda", dtype=torch.bool), at
    for _ in range(most - 1):
        want = choice.gather(1, last[:, None])
        hit = (parent == last[:, None]) & (token == want) & alive[:, None]
        alive = hit.any(1)
        last = torch.where(alive, hit.int().argmax(1), last)
        keep.append(torch.where(alive, last, -1))
    keep = torch.stack(keep, 1)
    n_keep = (keep >= 0).sum(1)
    base = st["lens"] - st["q_off"].diff()
    src, dst = base[:, None] + keep, (base[:, None] + torch.arange(most, device="cuda")).expand(s, most)
    live = keep >= 0
    row = torch.arange(s, device="cuda")[:, None].expand(s, most)[live]
    src, dst = src[live], dst[live]
    p, table = c["page"], st["table"].long()
    _move(st, table[row, src // p], src % p, table[row, dst // p], dst % p)
    return {"n_keep": n_keep.int(), "keep": keep.int(), "next": choice.gather(1, last[:, None])[:, 0], "len_out": (base + n_keep).int(),
            "k_pool": st["k_pool"], "v_pool": st["v_pool"]}


def _plain_beam(st):
    c = st["c"]
    g, b, k = c["n_group"], c["n_beam"], min(c["n_out"], c["n_vocab"])
    x = st["x"]
    top = x.amax(-1, keepdim=True)
    lse = top.double() + torch.log(torch.exp(x.double() - top.double()).sum(-1, keepdim=True))
    value, token = torch.sort(x, dim=-1, descending=True, stable=True)
    value, token = value[:, :k], token[:, :k]
    score = st["score"].double()[:, None] + (value.double() - lse)
    ended = st["ended"][:, None] != 0
    once = torch.where(torch.arange(k, device="cuda") == 0, st["score"].double()[:, None], -math.inf)
    score, token = torch.where(ended, once, score).reshape(g, -1), torch.where(ended, -1, token).reshape(g, -1)
    score, order = torch.sort(score, dim=-1, descending=True, stable=True)
    score, order = score[:, :c["n_out"]], order[:, :c["n_out"]]
    none = score == -math.inf
    row = torch.arange(g, device="cuda")[:, None] * b + order // k
    return {"score": score.float(), "row": torch.where(none, -1, row).int(), "token": torch.where(none, -1, token.gather(1, order)).int()}


def _plain_fork(st):
    c = st["c"]
    p, parent, table = c["page"], st["parent"].long(), st["table"]
    size = st["lens"][parent]
    whole = size // p
    col = torch.arange(table.shape[1], device="cuda")
    out = torch.where(col < whole[:, None], table[parent], torch.where(col == whole[:, None], st["fresh"][:, None], st["table_out"]))
    st["table_out"].copy_(out)
    st["len_out"].copy_(size)
    slot = torch.arange(p, device="cuda").expand(len(parent), p)
    part = slot < (size % p)[:, None]
    row = torch.arange(len(parent), device="cuda")[:, None].expand(-1, p)[part]
    slot = slot[part]
    _move(st, table[parent[row], whole[row].long()].long(), slot, st["fresh"][row].long(), slot)
    return {n: st[n] for n in ("len_out", "table_out", "k_pool", "v_pool")}


# ----------------------------------------------------------------------- work
def work(case):
    c = case
    if c["kind"] == "beam":
        n = c["n_group"] * c["n_beam"]
        return {"bytes": 4 * n * c["n_vocab"] + 8 * n + 12 * c["n_group"] * c["n_out"], "flops": 3 * n * c["n_vocab"]}
    if c["kind"] == "fork":
        rows = sum(n % c["page"] for n in _sizes(c))
        return {"bytes": 4 * rows * c["n_cache"] * c["n_kv"] * _row(c) + 8 * len(_sizes(c)) * (c["max_len"] // c["page"] + 3), "flops": 0}
    if c["kind"] == "keep":
        rows = sum(n - 1 for n in _kept(c))
        return {"bytes": 4 * rows * c["n_cache"] * c["n_kv"] * _row(c) + 12 * sum(_new(c)) + 4 * c["n_seq"] * (c["most"] + 5), "flops": 0}
    pre, w, rows, pairs = c["n_prefix"], c["window"], 0, 0
    low = pre
    for n, size in zip(_new(c), _lens(c)):
        first = pre + size - n                               # position of the first new token
        lo = max(0, first + 1 - w) if w else 0
        rows += pre + size - max(pre, lo)
        low = min(low, lo)
        pairs += n * (min(first, w - 1) if w else first) + n
    t = sum(_new(c))
    more = 4 * t * c["hd"] * (c["n_head"] + 4 * c["n_kv"]) if c["step"] else 0
    return {"bytes": 2 * (rows + max(0, pre - low)) * c["n_kv"] * _row(c) + 8 * t * c["n_head"] * c["hd"] + 4 * t * (-(-c["new"] // 32) + 1) + more,
            "flops": 4 * c["hd"] * c["n_head"] * pairs}


# ---------------------------------------------------------- 64-bit definition
def _row64(c, pool, pages, n, h, value):
    """Rows 0..n-1 of KV head h of the sequence with these pages, in 64 bits."""
    p, d = c["page"], c["hd"]
    at = torch.arange(n, device="cuda")
    pg, row = pages.long()[at // p], h * p + at % p
    if c["kv"] == "f16":
        return pool[pg, h, at % p].double()
    e = torch.arange(d, device="cuda")
    s, g, j, m, col = e // 32, e % 32 // 8, e % 8, e // 16, e % 16
    if c["kv"] == "q8_0":
        byte, low, base, size = (col * (d // 16) + m if value else g * (d // 4) + 8 * s + j), None, 128, d
    else:
        nib = m if value else (j >> 1) + 4 * (j & 1)
        byte, low, base, size = (col * (d // 32) if value else 4 * (g * (d // 32) + s)) + nib // 2, nib % 2, 8, d // 2
    b = pool[pg[:, None], row[:, None] * size + byte].int()
    b = b if low is None else (b >> (4 * low)) & 15
    at = c["n_kv"] * p * size + row[:, None] * (d // 16) + torch.arange(d // 16, device="cuda")
    sc = pool[pg[:, None], at].contiguous().view(torch.float16).double()
    return (b - base).double() * sc[:, s]


def _exact_tree(c, st):
    pre, grp, hd = c["n_prefix"], c["n_head"] // c["n_kv"], c["hd"]
    parent = st["parent"].tolist()
    paths, t = [], 0                                         # of every token, from the root
    for n in _new(c):
        for i in range(n):
            up = parent[t + i]
            paths.append((paths[t + up] if up >= 0 else []) + [i])
        t += n
    depth = torch.tensor([len(x) - 1 for x in paths], device="cuda")
    q, more = st["q"].double(), {}
    if c["step"]:
        first = torch.tensor([size - n for n, size in zip(_new(c), _lens(c)) for _ in range(n)], device="cuda")
        ang = (pre + first + depth).double()[:, None] * torch.exp(torch.arange(hd // 2, device="cuda", dtype=torch.float64) * (-2 * math.log(1e6) / hd))
        z = torch.polar(torch.ones_like(ang), ang)[:, None]

        def turned(x):
            y = torch.complex(x[..., :hd // 2], x[..., hd // 2:]) * z
            return torch.cat([y.real, y.imag], -1)

        q, k = turned(q), turned(st["k"].double())
        kp, vp, t = st["k_pool"].double(), st["v_pool"].double(), 0
        for s, (n, size) in enumerate(zip(_new(c), _lens(c))):
            for j in range(size - n, size):
                pg = int(st["table"][s, j // c["page"]])
                kp[pg, :, j % c["page"]], vp[pg, :, j % c["page"]] = k[t], st["v"][t].double()
                t += 1
        words = [[sum(1 << (j % 32) for j in x if j // 32 == w) for w in range(st["words"])] for x in paths]
        words = torch.tensor(words, device="cuda", dtype=torch.int64)
        more = {"mask": torch.where(words >= 2 ** 31, words - 2 ** 32, words).int(), "depth": depth.int(), "k": kp, "v": vp}
    out = torch.zeros_like(q)
    kp, vp = (st["k_pool"], st["v_pool"])
    if more:                                                 # attended as they are kept, rounded to halves
        kp, vp = more["k"].half(), more["v"].half()
    for h in range(c["n_kv"]):
        shared = [_row64(c, x, st["prefix"], pre, h, w == 1) for w, x in enumerate((kp, vp))]
        t = 0
        for s, (n, size) in enumerate(zip(_new(c), _lens(c))):
            k, v = (torch.cat([shared[w], _row64(c, x, st["table"][s], size, h, w == 1)]) for w, x in enumerate((kp, vp)))
            hidden = torch.zeros(n, pre + size, dtype=torch.bool)
            hidden[:, pre + size - n:] = True
            for i in range(n):
                hidden[i, [pre + size - n + j for j in paths[t + i]]] = False
                at = pre + size - n + len(paths[t + i]) - 1
                if c["window"]:
                    hidden[i, :min(pre + size - n, max(0, at + 1 - c["window"]))] = True
            for x in range(h * grp, (h + 1) * grp):
                y = q[t:t + n, x] @ k.T * hd ** -0.5
                y = c["cap"] * torch.tanh(y / c["cap"]) if c["cap"] else y
                out[t:t + n, x] = torch.softmax(y.masked_fill(hidden.cuda(), -math.inf), -1) @ v
            t += n
    return {"out": out} | more


def _exact_keep(c, st):
    parent, token, choice = (st[n].tolist() for n in ("parent", "token", "choice"))
    keep, nxt, t = [], [], 0
    for n in _new(c):
        path = [0]
        while len(path) < c["most"]:
            more = [j for j in range(n) if parent[t + j] == path[-1] and token[t + j] == choice[t + path[-1]]]
            if not more:
                break
            path.append(more[0])
        keep.append(path)
        nxt.append(choice[t + path[-1]])
        t += n
    pools = {"k_pool": st["k_pool"].clone(), "v_pool": st["v_pool"].clone()}
    p = c["page"]
    for s, (path, n, size) in enumerate(zip(keep, _new(c), _lens(c))):
        pages = st["table"][s].tolist()
        for k, j in enumerate(path):
            a, b = size - n + j, size - n + k
            for name, pool in pools.items():
                for x, y in zip(_runs(c, pool), _runs(c, st[name])):
                    x[:, pages[b // p], :, b % p] = y[:, pages[a // p], :, a % p]
    if c["kv"] == "f16":
        pools = {n: x.double() for n, x in pools.items()}
    return {"n_keep": _ints([len(x) for x in keep]), "keep": _ints([x + [-1] * (c["most"] - len(x)) for x in keep]), "next": _ints(nxt),
            "len_out": _ints([size - n + len(x) for x, n, size in zip(keep, _new(c), _lens(c))])} | pools


def _exact_beam(c, st):
    score, row, token = [], [], []
    for g in range(c["n_group"]):
        own_rows = slice(g * c["n_beam"], (g + 1) * c["n_beam"])
        s, x = st["score"][own_rows].double(), st["x"][own_rows].double()
        flat = s[:, None] + torch.log_softmax(x, -1)
        for b in torch.nonzero(st["ended"][own_rows]).flatten().tolist():
            flat[b] = -math.inf
            flat[b, 0] = s[b]
        best = torch.topk(flat.flatten(), min(flat.numel(), c["n_out"]))
        pairs = sorted(zip((-best.values).tolist(), best.indices.tolist()))
        found = [(-v, i // c["n_vocab"], i % c["n_vocab"]) for v, i in pairs if v < math.inf]
        done = st["ended"][own_rows].tolist()
        found += [(-math.inf, None, None)] * (c["n_out"] - len(found))
        score.append([v for v, _, _ in found])
        row.append([-1 if b is None else g * c["n_beam"] + b for _, b, _ in found])
        token.append([-1 if b is None or done[b] else i for _, b, i in found])
    return {"score": torch.tensor(score, dtype=torch.float64, device="cuda"), "row": _ints(row), "token": _ints(token)}


def _exact_fork(c, st):
    lens, table, out, fresh = st["lens"].tolist(), st["table"].tolist(), st["table_out"].tolist(), st["fresh"].tolist()
    pools = {"k_pool": st["k_pool"].clone(), "v_pool": st["v_pool"].clone()}
    parent = st["parent"].tolist()
    for i, up in enumerate(parent):
        whole, part = divmod(lens[up], c["page"])
        out[i][:whole] = table[up][:whole]
        out[i][whole] = fresh[i]
        for name, pool in pools.items():
            for x, y in zip(_runs(c, pool), _runs(c, st[name])):
                if part:
                    x[:, fresh[i], :, :part] = y[:, table[up][whole], :, :part]
    if c["kv"] == "f16":
        pools = {n: x.double() for n, x in pools.items()}
    return {"len_out": _ints([lens[up] for up in parent]), "table_out": _ints(out)} | pools


def exact(case, seed):
    st = prepare(case, seed)
    return {"tree": _exact_tree, "keep": _exact_keep, "beam": _exact_beam, "fork": _exact_fork}[case["kind"]](case, st)
