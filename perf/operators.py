"""The paged key/value cache's operators as runnable cases.

A batch of sequences is served together: their keys and values live in pages of
one pool, new rows are rotated and appended for all sequences in one call, and
the attention over the pages takes single tokens, prompt chunks and mixtures of
both, with a tanh cap on the scores, a sliding window, and a prefix that all
sequences share.  `listed()` names the cases, `draw()` makes others of the same
ranges, `prepare()` makes a case's inputs on the GPU, and `run()` is one pass:
in elementary torch operations, or, with `own` set, through the public entry
points of g4run_amd.  `exact()` computes the same values in 64 bits.

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
LARGEST = 8 * 1024 * 32 * 4 * 256          # key elements of the largest drawn batch
MOST = 6 * 10 ** 9                         # (head, token, key) products of the largest drawn batch, by element


def listed():
    gemma = dict(n_head=8, n_kv=4, hd=256)     # the synthetic decoder's heads
    wide = dict(n_head=32, n_kv=8, hd=128)
    return [
        # one sequence's next token into a long cache: call and launch latency
        _append("append_one_f16", "f16", n_seq=1, max_len=8191, **gemma),
        # the next token of 64 short conversations, 8-bit cache
        _append("append_batch_q8_0", "q8_0", n_seq=64, max_len=96, page=16, **wide),
        # three ragged prompts (2048, 1659, ... tokens) with padded rows behind
        _append("append_prompts_f16", "f16", n_seq=3, max_len=2600, new=2048, pad=13, page=64, **gemma),
        # one sequence's token over a short cache: latency
        _attn("attn_one_f16", "f16", n_seq=1, max_len=100, **gemma),
        # 32 conversations of up to 8192 positions, one token each: bandwidth
        _attn("attn_decode_f16", "f16", n_seq=32, max_len=8192, page=64, **gemma),
        # 64 conversations over 8-bit pages, capped scores
        _attn("attn_decode_q8_0_cap", "q8_0", n_seq=64, max_len=4096, cap=50.0, **wide),
        # sliding-window layers of wide heads over 4-bit pages
        _attn("attn_decode_q4_0_window", "q4_0", n_seq=16, max_len=5000, window=1024, page=16, n_head=8, n_kv=2, hd=512),
        # prompt chunks of four sequences behind cached positions, capped scores
        _attn("attn_prompts_f16_cap", "f16", n_seq=4, max_len=4300, new=509, cap=30.0, pad=3, **gemma),
        # two prompt chunks among thirty single tokens, small heads
        _attn("attn_mixed_f16", "f16", n_seq=32, max_len=2000, new=300, mix=2, n_head=16, n_kv=4, hd=64),
        # four answers drawn from one short prompt
        _attn("prefix_few_f16", "f16", n_seq=4, max_len=70, n_prefix=1001, **gemma),
        # 64 conversations behind one long system prompt
        _attn("prefix_batch_f16", "f16", n_seq=64, max_len=512, n_prefix=8192, page=64, **gemma),
        # the same over 8-bit pages, two new tokens at most (a verified draft)
        _attn("prefix_batch_q8_0", "q8_0", n_seq=24, max_len=300, new=2, n_prefix=16383, **wide),
    ]


def _append(name, kv, **more):
    c = dict(kind="append", kv=kv, page=32, new=1, mix=0, pad=0, n_prefix=0, n_rot=more["hd"], interleaved=False, base=1e6)
    return ({"name": name} if name else {}) | c | more


def _attn(name, kv, **more):
    c = dict(kind="attn", kv=kv, page=32, new=1, mix=0, pad=0, n_prefix=0, cap=0.0, window=0)
    return ({"name": name} if name else {}) | c | more


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kv, page = rng.choice(["f16", "f16", "q8_0", "q4_0"]), rng.choice([16, 32, 48, 64, 128])
    hd = rng.choice([64, 128, 128, 256, 256, 512])
    n_kv = rng.choice([1, 2, 4, 8] if hd < 512 else [1, 2])
    n_head = n_kv * rng.choice([1, 2, 3, 4, 8, 12] if hd < 512 else [1, 2, 4, 8])
    head = dict(n_head=n_head, n_kv=n_kv, hd=hd, page=page)
    kind = rng.choice(["append", "append", "decode", "decode", "chunk", "chunk", "prefix", "prefix"])
    if kind == "append":
        new = rng.choice([1, _log(rng, 2, 1024)])
        n_seq = _log(rng, 1, min(64, max(1, 4096 * 16 * 256 // (new * (n_head + 2 * n_kv) * hd))))
        return _append(None, kv, n_seq=n_seq, new=new, max_len=new + _log(rng, 1, 400), pad=rng.choice([0, 0, 5]) if new > 1 else 0,
                       n_prefix=rng.choice([0, 0, 100000]), **head) | dict(n_rot=rng.choice([hd, hd, hd // 2]), interleaved=rng.random() < 0.3,
                                                                           base=rng.choice([1e4, 1e6]))
    cap, window = rng.choice([0.0, 0.0, 30.0, 50.0]), rng.choice([0, 0, 512])
    n_seq = _log(rng, 1, 64)
    most = LARGEST // (n_seq * n_kv * hd)
    if kind == "decode":
        return _attn(None, kv, n_seq=n_seq, max_len=_log(rng, 1, min(16384, max(2, most))), cap=cap, window=window, **head)
    if kind == "chunk":
        new = _log(rng, 2, max(3, min(509, 16384 // (n_seq * (n_head // 8 + 1)))))
        behind = max(2, min(4000, most // 4, MOST // (n_seq * new * n_head * hd)))
        return _attn(None, kv, n_seq=n_seq, max_len=new + _log(rng, 1, behind), new=new, mix=rng.choice([0, 1]), cap=cap, window=window, **head)
    shared = max(21, min(16384, most, MOST // (n_seq * n_head * hd)))
    return _attn(None, kv, n_seq=n_seq, max_len=_log(rng, 1, min(600, max(2, most // 2))), n_prefix=_log(rng, 20, shared), cap=cap, **head)


# ------------------------------------------------------------------ the batch
def _frac(i):
    return (0.5 + 0.6180339887498949 * i) % 1.0


def _new(c):
    """New tokens of each sequence: the first has the most; of a mixed batch
    only the first `mix` sequences have more than one."""
    return [c["new"] if i == 0 else 1 + int((c["new"] - 1) * _frac(i)) if not c["mix"] or i < c["mix"] else 1 for i in range(c["n_seq"])]


def _lens(c):
    """Positions in each sequence's own pages, its new tokens included."""
    return [c["max_len"] if i == 0 else n + int((c["max_len"] - n) * _frac(i + 7)) for i, n in enumerate(_new(c))]


def _row(c):
    """Bytes of one cached row."""
    return c["hd"] * 2 if c["kv"] == "f16" else c["hd"] // (1 if c["kv"] == "q8_0" else 2) + c["hd"] // 16


def _pool(c, n_pages, gen):
    """A pool of n_pages whose rows hold values of unit size."""
    h, p, d = c["n_kv"], c["page"], c["hd"]
    if c["kv"] == "f16":
        return torch.randn(n_pages, h, p, d, device="cuda", generator=gen, dtype=torch.float16)
    sc = torch.rand(n_pages, h * p * (d // 32), device="cuda", generator=gen) * 0.5 + 0.75
    if c["kv"] == "q8_0":
        q = torch.randn(n_pages, h * p * d, device="cuda", generator=gen, dtype=torch.float16) * 42
        q, sc = q.clamp_(-127, 127).round_().add_(128).to(torch.uint8), (sc / 42).half()
    else:
        q = torch.randn(2, n_pages, h * p * d // 2, device="cuda", generator=gen, dtype=torch.float16) * 2.6
        q = q.clamp_(-8, 7).round_().add_(8).to(torch.uint8)
        q = q[0] | (q[1] << 4)
        sc = (sc / -2.6).half()
    return torch.cat([q, sc.view(torch.uint8)], 1)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    new, lens = _new(c), _lens(c)
    n_new = sum(new)
    n_tok = n_new + c["pad"]
    pages = [-(-n // c["page"]) for n in lens]
    n_pre = -(-c["n_prefix"] // c["page"]) if c["kind"] == "attn" else 0
    order = torch.randperm(sum(pages) + n_pre + 3, generator=host).to(torch.int32)
    table = torch.full((c["n_seq"], max(pages)), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = order[at:at + n]
        at += n
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    q_off = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32)
    st = dict(c=c, n_new=n_new, n_tok=n_tok, most_new=max(new), lens=torch.tensor(lens, dtype=torch.int32).cuda(), table=table.cuda(), q_off=q_off.cuda(),
              prefix=order[at:at + n_pre].cuda(), k_pool=_pool(c, len(order), gen), v_pool=_pool(c, len(order), gen),
              q=rand(n_tok, c["n_head"], c["hd"]) * 1.5, out=rand(n_tok, c["n_head"], c["hd"]), kept={})
    if c["kind"] == "append":
        st["k"], st["v"] = rand(n_tok, c["n_kv"], c["hd"]), rand(n_tok, c["n_kv"], c["hd"])
        for n in ("k_read", "v_read"):
            st[n] = torch.zeros(n_new, c["n_kv"], c["hd"], device="cuda", dtype=torch.float16)
    return st


def run(state):
    if own:
        return _own_append(state) if state["c"]["kind"] == "append" else _own_attn(state)
    return _plain_append(state) if state["c"]["kind"] == "append" else _plain_attn(state)


# ---------------------------------------------- the library's own entry points
def _plan(st):
    """The cache, the batch's description and the workspace, which a serving
    loop keeps from call to call."""
    if not st["kept"]:
        import g4run_amd as G
        G.init()
        c = st["c"]
        kv = G.PagedKV(TYPES[c["kv"]], c["n_kv"], c["hd"], c["page"], st["k_pool"].shape[0], k=st["k_pool"].data_ptr(), v=st["v_pool"].data_ptr())
        one = c["new"] == 1 and not c["pad"]
        batch = G.PagedBatch(c["n_seq"], st["n_tok"], st["lens"].data_ptr(), st["table"].data_ptr(), st["table"].shape[1], c["max_len"],
                             q_off=None if one else st["q_off"].data_ptr(), n_prefix=c["n_prefix"],
                             prefix=st["prefix"].data_ptr() if len(st["prefix"]) else None)
        st["kept"] = dict(G=G, kv=kv, batch=batch)
        if c["kind"] == "append":
            st["kept"]["rope"] = G.Rope(c["n_rot"], c["base"], interleaved=c["interleaved"])
        else:
            st["kept"]["ws"] = G.Buffer(max(16, G.paged_attn_workspace_bytes(kv, batch, c["n_head"])))
    return st["kept"]


def _own_append(st):
    p, c = _plan(st), st["c"]
    p["G"].paged_append(p["kv"], p["batch"], st["k"].data_ptr(), st["v"].data_ptr(), q=st["q"].data_ptr(), q_out=st["out"].data_ptr(),
                        n_head=c["n_head"], rope=p["rope"])
    if c["kv"] == "f16":
        return {"q": st["out"], "k": st["k_pool"], "v": st["v_pool"]}
    p["G"].paged_read(p["kv"], p["batch"], st["k_read"].data_ptr(), st["v_read"].data_ptr(), out_type=TYPES["f16"])
    return {"q": st["out"], "k": st["k_read"], "v": st["v_read"]}


def _own_attn(st):
    p, c = _plan(st), st["c"]
    p["G"].paged_attn(p["kv"], p["batch"], st["q"].data_ptr(), c["n_head"], st["out"].data_ptr(), scale=c["hd"] ** -0.5, softcap=c["cap"],
                      window=c["window"], ws=p["ws"])
    return st["out"]


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


def _slots(st):
    """Sequence and position in its own pages of every new token."""
    tok = torch.arange(st["n_new"], device="cuda")
    seq = torch.searchsorted(st["q_off"][1:].long(), tok, right=True)
    return seq, tok - st["q_off"][seq + 1] + st["lens"][seq]


def _plain_attn(st):
    c, hd, grp = st["c"], st["c"]["hd"], st["c"]["n_head"] // st["c"]["n_kv"]
    s, n, pre = c["n_seq"], st["most_new"], c["n_prefix"]
    at = torch.arange(n, device="cuda")
    q = st["q"][(st["q_off"][:-1, None] + at).clamp(max=st["n_tok"] - 1).long()]             # [seq, new, head, hd]
    q = q.reshape(s, n, c["n_kv"], grp, hd).permute(0, 2, 3, 1, 4).reshape(s, c["n_kv"], grp * n, hd)
    k, v = (_dense(c, st[p], st["table"], p == "v_pool") for p in ("k_pool", "v_pool"))
    sc = q @ k.transpose(-1, -2)
    if pre:
        kp, vp = (_dense(c, st[p], st["prefix"][None], p == "v_pool")[0, :, :pre] for p in ("k_pool", "v_pool"))
        qp = q.transpose(0, 1).reshape(c["n_kv"], -1, hd)
        sc = torch.cat([(qp @ kp.transpose(-1, -2)).reshape(c["n_kv"], s, grp * n, pre).transpose(0, 1), sc], -1)
    sc = sc * hd ** -0.5
    if c["cap"]:
        sc = c["cap"] * torch.tanh(sc / c["cap"])
    pos = (pre + st["lens"] - st["q_off"].diff())[:, None] + at                               # [seq, new]
    key = torch.arange(sc.shape[-1], device="cuda")
    seen = key <= pos[..., None]
    if c["window"]:
        seen &= key > pos[..., None] - c["window"]
    sc = sc.reshape(s, c["n_kv"], grp, n, -1).masked_fill(~seen[:, None, None], -math.inf).reshape(sc.shape)
    e = torch.exp(sc - sc.amax(-1, keepdim=True).clamp(min=-3e38))
    o = e[..., pre:] @ v
    if pre:
        o += (e[..., :pre].transpose(0, 1).reshape(c["n_kv"], -1, pre) @ vp).reshape(c["n_kv"], s, grp * n, hd).transpose(0, 1)
    o = o / e.sum(-1, keepdim=True).clamp(min=1e-30)
    seq, _ = _slots(st)
    tok = torch.arange(st["n_new"], device="cuda")
    o = o.reshape(s, c["n_head"], n, hd)[seq, :, tok - st["q_off"][seq]]
    return torch.cat([o, st["out"][st["n_new"]:]])


def _turn(c, x, cos, sin):
    r = c["n_rot"]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if c["interleaved"] else (x[..., :r // 2], x[..., r // 2:r])
    t = (a * cos - b * sin, b * cos + a * sin)
    return torch.cat([torch.stack(t, -1).flatten(-2) if c["interleaved"] else torch.cat(t, -1), x[..., r:]], -1)


def _blocks(c, x):
    """Rows of values as (quants, scales) of blocks of 32."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    if c["kv"] == "q8_0":
        top = b.abs().amax(-1, keepdim=True)
        return torch.round(b * torch.where(top > 0, 127 / top, 0)) + 128, top * (1 / 127)
    top = b.gather(-1, b.abs().argmax(-1, keepdim=True))
    d = top * -0.125
    return torch.trunc(b * torch.where(d != 0, 1 / d, 0) + 8.5).clamp(max=15), d


def _put(c, pool, page, slot, x, value):
    """Rows [token, n_kv, hd] into their pages."""
    h, p, d = c["n_kv"], c["page"], c["hd"]
    head = torch.arange(h, device="cuda")
    if c["kv"] == "f16":
        pool[page[:, None], head, slot[:, None]] = x.half()
        return
    q, sc = _blocks(c, x)
    q, t = q.to(torch.uint8), x.shape[0]
    n = h * p * d // (1 if c["kv"] == "q8_0" else 2)
    if value:
        q = q.reshape(t, h, d // 16, 16).transpose(-1, -2)
    else:
        q = q.reshape(t, h, d // 32, 4, 8).transpose(-2, -3)
        if c["kv"] == "q4_0":
            q = q.reshape(t, h, 4, d // 32, 4, 2).transpose(-1, -2)
    q = q.reshape(t, h, -1)
    if c["kv"] == "q4_0":
        q = q[..., 0::2] | (q[..., 1::2] << 4)
    row = head * p + slot[:, None]
    w = q.shape[-1]
    pool[page[:, None, None], row[..., None] * w + torch.arange(w, device="cuda")] = q
    sc = sc.half().reshape(t, h, d // 32).view(torch.uint8)
    pool[page[:, None, None], n + row[..., None] * (d // 16) + torch.arange(d // 16, device="cuda")] = sc


def _plain_append(st):
    c, n = st["c"], st["n_new"]
    seq, own_pos = _slots(st)
    freq = c["base"] ** (-2 * torch.arange(c["n_rot"] // 2, device="cuda", dtype=torch.float64) / c["n_rot"])
    ang = (c["n_prefix"] + own_pos).double()[:, None, None] * freq
    cos, sin = torch.cos(ang).float(), torch.sin(ang).float()
    page, slot = st["table"][seq, own_pos // c["page"]].long(), own_pos % c["page"]
    q = torch.cat([_turn(c, st["q"][:n], cos, sin), st["out"][n:]])
    _put(c, st["k_pool"], page, slot, _turn(c, st["k"][:n], cos, sin), False)
    _put(c, st["v_pool"], page, slot, st["v"][:n], True)
    if c["kv"] == "f16":
        return {"q": q, "k": st["k_pool"], "v": st["v_pool"]}
    back = lambda p, value: _values(c, st[p][page], value)[torch.arange(n, device="cuda"), :, slot].half()  # noqa: E731
    return {"q": q, "k": back("k_pool", False), "v": back("v_pool", True)}


# ----------------------------------------------------------------------- work
def _seen(c):
    """(rows of keys read, (token, key) pairs) of a pass, for one KV head."""
    pre, w, rows, pairs = c["n_prefix"], c["window"], 0, 0
    low = pre
    for n, size in zip(_new(c), _lens(c)):
        first = pre + size - n                               # position of the first new token
        lo = max(0, first + 1 - w) if w else 0
        rows += pre + size - max(pre, lo)
        low = min(low, lo)
        pairs += sum(min(first + i + 1, w or first + i + 1) for i in range(n))
    return rows + max(0, pre - low), pairs


def work(case):
    c, t = case, sum(_new(case))
    if c["kind"] == "append":
        return {"bytes": t * c["hd"] * 4 * (2 * c["n_head"] + 2 * c["n_kv"]) + 2 * t * c["n_kv"] * _row(c),
                "flops": 6 * t * c["n_rot"] // 2 * (c["n_head"] + c["n_kv"])}
    rows, pairs = _seen(c)
    return {"bytes": 2 * rows * c["n_kv"] * _row(c) + 8 * t * c["n_head"] * c["hd"], "flops": 4 * c["hd"] * c["n_head"] * pairs}


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


def _exact_attn(c, st):
    pre, grp = c["n_prefix"], c["n_head"] // c["n_kv"]
    out = st["out"].double()
    for h in range(c["n_kv"]):
        shared = [_row64(c, st[p], st["prefix"], pre, h, p == "v_pool") for p in ("k_pool", "v_pool")]
        t = 0
        for i, (n, size) in enumerate(zip(_new(c), _lens(c))):
            k, v = (torch.cat([shared[w], _row64(c, st[p], st["table"][i], size, h, w == 1)]) for w, p in enumerate(("k_pool", "v_pool")))
            at = torch.arange(pre + size - n, pre + size, device="cuda")[:, None]
            j = torch.arange(pre + size, device="cuda")
            hidden = (j > at) | ((j <= at - c["window"]) if c["window"] else False)
            for q in range(h * grp, (h + 1) * grp):
                s = st["q"][t:t + n, q].double() @ k.T * c["hd"] ** -0.5
                s = c["cap"] * torch.tanh(s / c["cap"]) if c["cap"] else s
                out[t:t + n, q] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ v
            t += n
    return out


def _exact_append(c, st):
    half = c["n_rot"] // 2
    pos = torch.cat([c["n_prefix"] + torch.arange(s - n, s, dtype=torch.float64) for n, s in zip(_new(c), _lens(c))]).cuda()
    ang = pos[:, None] * torch.exp(torch.arange(half, device="cuda", dtype=torch.float64) * (-2 * math.log(c["base"]) / c["n_rot"]))
    z = torch.polar(torch.ones_like(ang), ang)[:, None]
    a = torch.arange(half, device="cuda") * (2 if c["interleaved"] else 1)
    b = a + (1 if c["interleaved"] else half)

    def turned(x):
        x = x[:st["n_new"]].double()
        y = torch.complex(x[..., a], x[..., b]) * z
        x[..., a], x[..., b] = y.real, y.imag
        return x

    def stored(x):
        if c["kv"] == "f16":
            return x
        w = x.unflatten(-1, (-1, 32))
        if c["kv"] == "q8_0":
            top = w.abs().amax(-1, keepdim=True)
            y = torch.round(w * 127 / top.clamp(min=1e-300)) * (top / 127).half().double()
        else:
            d = w.gather(-1, w.abs().argmax(-1, keepdim=True)) / -8
            y = ((w / torch.where(d == 0, 1, d) + 8.5).floor().clamp(max=15) - 8) * d.half().double()
        return y.reshape(x.shape)

    q, k, v = st["out"].double(), stored(turned(st["k"])), stored(st["v"][:st["n_new"]].double())
    q[:st["n_new"]] = turned(st["q"])
    if c["kv"] != "f16":
        return {"q": q, "k": k, "v": v}
    pools, t = {"k": st["k_pool"].double(), "v": st["v_pool"].double()}, 0
    for i, (n, size) in enumerate(zip(_new(c), _lens(c))):
        for j in range(size - n, size):
            pg = int(st["table"][i, j // c["page"]])
            pools["k"][pg, :, j % c["page"]], pools["v"][pg, :, j % c["page"]] = k[t], v[t]
            t += 1
    return {"q": q, **pools}


def exact(case, seed):
    st = prepare(case, seed)
    return _exact_append(case, st) if case["kind"] == "append" else _exact_attn(case, st)
