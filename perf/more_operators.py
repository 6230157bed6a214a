"""The operators for drafted trees and branching sequences over a paged f16 KV cache, as workloads that are timed and checked.

Kinds of case, and what they stand for:
  plan  `tree_step`: the positions and ancestor masks of a step's drafted trees, from each node's parent
  attn  `attn_paged_tree`: attention of the trees' nodes over the pages, with or without a prefix that all of the batch shares
  keep  `tree_accept`, `kv_rows_move`, `kv_pages_fork` in a row: which drafted path the choices confirm, its keys and values
        moved to where the sequence goes on (every layer), the pages behind it given back
  fork  `kv_pages_fork`, `kv_rows_move`: beams of several requests that go on from others of the same request: full pages
        shared, the last one copied (every layer), pages that nobody holds any more given back
  logp  `logits_logprobs`: log probabilities of given tokens with their ranks, the entropy and the likeliest alternatives

`own` false computes them plainly in torch, true through the backend. Lengths and trees' sizes follow from a case's values
alone; the data, the trees' shapes and where pages lie from the seed.
"""
import math
import random

import numpy as np
import torch

own = False
DEV = "cuda"
_HIP = None


def _hip():
    """The program's one backend context."""
    global _HIP
    if _HIP is None:
        from rustingstrata_amd.backend import HipBackend
        _HIP = HipBackend(0)
    return _HIP


# ---- the cases ----
def listed():
    return [
        # one user's step: a small fixed tree
        {"name": "plan_1", "kind": "plan", "nseq": 1, "lo": 26, "hi": 26, "min_len": 500, "max_len": 600, "words": 1, "mix": 1},
        # a full server's step, trees of all sizes
        {"name": "plan_512", "kind": "plan", "nseq": 512, "lo": 1, "hi": 64, "min_len": 1, "max_len": 8000, "words": 2, "mix": 2},
        # one user's tree over a chat turn
        {"name": "attn_1", "kind": "attn", "nseq": 1, "lo": 16, "hi": 16, "min_len": 900, "max_len": 1000, "prefix": 0, "page": 64, "nh": 32, "nkv": 4, "hd": 128, "win": 0, "sink": 0, "gate": 0, "words": 1, "mix": 3},
        # a batch with contexts and trees of very different sizes
        {"name": "attn_32", "kind": "attn", "nseq": 32, "lo": 4, "hi": 20, "min_len": 100, "max_len": 9000, "prefix": 0, "page": 16, "nh": 32, "nkv": 4, "hd": 128, "win": 0, "sink": 0, "gate": 0, "words": 1, "mix": 4},
        # a system prompt that all share, small heads, sink logits and output gates
        {"name": "attn_prefix_24", "kind": "attn", "nseq": 24, "lo": 3, "hi": 13, "min_len": 1, "max_len": 700, "prefix": 6001, "page": 32, "nh": 16, "nkv": 8, "hd": 64, "win": 0, "sink": 1, "gate": 1, "words": 1, "mix": 5},
        # wide trees over long documents
        {"name": "attn_wide_8", "kind": "attn", "nseq": 8, "lo": 64, "hi": 64, "min_len": 6000, "max_len": 30000, "prefix": 0, "page": 64, "nh": 32, "nkv": 4, "hd": 128, "win": 0, "sink": 0, "gate": 0, "words": 2, "mix": 6},
        # the end of one user's step
        {"name": "keep_1", "kind": "keep", "nseq": 1, "lo": 26, "hi": 26, "min_len": 500, "max_len": 600, "page": 64, "nkv": 4, "hd": 128, "caches": 96, "path": 8, "words": 1, "mix": 7},
        # the end of a full server's step
        {"name": "keep_256", "kind": "keep", "nseq": 256, "lo": 4, "hi": 64, "min_len": 50, "max_len": 300, "page": 32, "nkv": 4, "hd": 128, "caches": 24, "path": 12, "words": 2, "mix": 8},
        # one request's beams
        {"name": "fork_5", "kind": "fork", "requests": 1, "beams": 5, "min_len": 700, "max_len": 1000, "page": 64, "nkv": 4, "hd": 128, "caches": 96, "mix": 9},
        # beams of many requests
        {"name": "fork_256", "kind": "fork", "requests": 32, "beams": 8, "min_len": 100, "max_len": 1200, "page": 64, "nkv": 4, "hd": 128, "caches": 24, "mix": 10},
        # one choice reported with its alternatives
        {"name": "logp_1", "kind": "logp", "rows": 1, "n": 151936, "m": 1, "k": 5, "mask": 0, "mix": 11},
        # a prompt scored token by token
        {"name": "logp_1001", "kind": "logp", "rows": 1001, "n": 151936, "m": 1, "k": 20, "mask": 0, "mix": 12},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "attn", "attn", "attn", "keep", "fork", "logp", "logp"])
    mix, page = rng.randrange(1 << 20), rng.choice([16, 32, 64, 128])
    if kind == "logp":
        return {"kind": kind, "rows": _log(rng, 1, 1001), "n": rng.choice([_log(rng, 1000, 151936), 151936]), "m": rng.randrange(0, 5), "k": rng.choice([0, 1, 5, 20, rng.randrange(1, 65)]), "mask": rng.choice([0, 0, 1]), "mix": mix}
    hi = rng.choice([rng.randrange(1, 9), rng.randrange(2, 33), rng.randrange(33, 65)])
    tree = {"nseq": _log(rng, 1, 512 if kind == "plan" else 128 if kind == "keep" else 40), "lo": rng.randrange(1, hi + 1), "hi": hi, "words": -(-hi // 32) + rng.choice([0, 0, 1]), "mix": mix}
    if kind == "plan":
        return {"kind": kind, "min_len": 1, "max_len": _log(rng, 10, 8000)} | tree
    if kind == "keep":
        return {"kind": kind, "min_len": 1, "max_len": _log(rng, 10, 400), "page": page, "nkv": rng.choice([1, 4, 8]), "hd": rng.choice([64, 128]), "caches": rng.choice([2, 8, 20]), "path": rng.randrange(1, 13)} | tree
    if kind == "fork":
        return {"kind": kind, "requests": _log(rng, 1, 24), "beams": rng.randrange(1, 9), "min_len": 1, "max_len": _log(rng, 20, 1200), "page": page, "nkv": rng.choice([1, 4, 8]), "hd": rng.choice([64, 128]), "caches": rng.choice([2, 8, 16]), "mix": mix}
    nh, nkv, hd = rng.choice([(32, 4, 128), (32, 4, 128), (32, 8, 128), (16, 8, 64), (16, 16, 128), (16, 2, 64)])
    return {"kind": kind, "min_len": 1, "max_len": _log(rng, 60, 6000), "prefix": rng.choice([0, 0, _log(rng, 100, 6000)]), "page": page, "nh": nh, "nkv": nkv, "hd": hd,
            "win": rng.choice([0, 0, 0, 1024]), "sink": rng.choice([0, 0, 1]), "gate": rng.choice([0, 0, 1])} | tree


# ---- sizes: what a case's values alone say ----
def _sizes(c):
    """(nodes, cached tokens before them) of each sequence."""
    r = random.Random(c["mix"])
    return [r.randint(c["lo"], c["hi"]) for _ in range(c["nseq"])], [_log(r, c["min_len"], c["max_len"]) for _ in range(c["nseq"])]


def _beams(c):
    """Cached tokens of each request's shared prompt and of each of its beams, prompt included."""
    r = random.Random(c["mix"])
    prompt = [_log(r, c["min_len"], c["max_len"]) for _ in range(c["requests"])]
    return prompt, [p + 1 + r.randrange(40) for p in prompt for _ in range(c["beams"])]


# ---- inputs ----
def _gen(seed, part):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1009 + part) % (1 << 62))
    return g


def _randn(seed, part, *shape, dtype=torch.float32):
    return torch.randn(*shape, device=DEV, dtype=dtype, generator=_gen(seed, part))


def _i32(v):
    return torch.tensor(np.asarray(v), device=DEV, dtype=torch.int32)


def _zeros(*shape, dtype=torch.int32):
    return torch.zeros(*shape, device=DEV, dtype=dtype)


def _cdiv(a, b):
    return -(-a // b)


def _parents(rng, sizes):
    """A drafted tree for each sequence: row 0 its root, a node's parent before it, wide near the root."""
    return np.concatenate([np.concatenate([[-1], (np.arange(1, n) * rng.random(n - 1) ** 2).astype(np.int64)]) for n in sizes]).astype(np.int32)


def _depths(parent, q_start):
    depth = np.zeros(len(parent), dtype=np.int64)
    for s in range(len(q_start) - 1):
        for r in range(q_start[s] + 1, q_start[s + 1]):
            depth[r] = depth[q_start[s] + parent[r]] + 1
    return depth


def _masks(parent, q_start, words):
    bits = np.zeros((len(parent), words), dtype=np.uint32)
    for s in range(len(q_start) - 1):
        for i in range(q_start[s + 1] - q_start[s]):
            r = q_start[s] + i
            if parent[r] >= 0:
                bits[r] = bits[q_start[s] + parent[r]]
            bits[r, i // 32] |= np.uint32(1 << (i % 32))
    return bits.view(np.int32)


def _tables(rng, lengths, page, spare=0):
    """Block tables of sequences whose pages lie anywhere in a pool, the unused pages, and the pool's size."""
    need = [_cdiv(n, page) for n in lengths]
    n_pages = sum(need) + spare + 1
    order = rng.permutation(n_pages).astype(np.int32)
    tables = np.zeros((len(lengths), max(need + [1])), dtype=np.int32)
    at = 0
    for s, k in enumerate(need):
        tables[s, :k] = order[at:at + k]
        at += k
    return tables, order[at:], n_pages


class _State:
    pass


def prepare(case, seed):
    s = _State()
    s.c = case
    {"plan": _prepare_plan, "attn": _prepare_attn, "keep": _prepare_keep, "fork": _prepare_fork, "logp": _prepare_logp}[case["kind"]](s, case, seed)
    return s


def _prepare_trees(s, c, seed):
    s.rng = np.random.default_rng(int(seed))
    s.q, s.before = _sizes(c)
    s.starts = np.concatenate([[0], np.cumsum(s.q)])
    s.t = int(s.starts[-1])
    s.parents = _parents(s.rng, s.q)
    s.parent, s.q_start, s.len = _i32(s.parents), _i32(s.starts), _i32([b + n for b, n in zip(s.before, s.q)])


def _prepare_plan(s, c, seed):
    _prepare_trees(s, c, seed)
    s.prefix_len = _i32([int(seed) % 5000])
    s.pos, s.mask = _zeros(s.t), _zeros(s.t, c["words"])


def _prepare_attn(s, c, seed):
    _prepare_trees(s, c, seed)
    nh, nkv, hd, page, P = c["nh"], c["nkv"], c["hd"], c["page"], c["prefix"]
    length = [b + n for b, n in zip(s.before, s.q)]
    tables, _, s.n_pages = _tables(s.rng, length + [P], page)
    s.max_pages, s.max_q = max(1, max(_cdiv(n, page) for n in length)), max(s.q)
    s.prefix = _i32(tables[-1, :max(1, _cdiv(P, page))])
    s.tables = _i32(tables[:-1, :s.max_pages])
    s.pos = _i32(P + np.repeat(s.before, s.q) + _depths(s.parents, s.starts))
    s.mask = _i32(_masks(s.parents, s.starts, c["words"]))
    s.prefix_len = _i32([P])
    s.x = 1.5 * _randn(seed, 1, s.t, nh, hd)
    s.kc = _randn(seed, 2, s.n_pages * page, nkv, hd).to(torch.float16)
    s.vc = (0.5 * _randn(seed, 3, s.n_pages * page, nkv, hd)).to(torch.float16)
    s.sink = _randn(seed, 4, nh) if c["sink"] else None
    s.gate = _randn(seed, 5, s.t, nh, 2, hd) if c["gate"] else None
    s.out = torch.zeros_like(s.x)


def _caches(s, c, seed):
    """The K and V caches of all layers, and their addresses as the program hands them over."""
    s.n_slots, s.width = s.n_pages * c["page"], c["nkv"] * c["hd"]
    s.kv = _randn(seed, 2, c["caches"], s.n_slots, s.width, dtype=torch.float16)
    s.addresses = torch.tensor([s.kv[i].data_ptr() for i in range(c["caches"])], device=DEV, dtype=torch.int64)


def _prepare_keep(s, c, seed):
    _prepare_trees(s, c, seed)
    page = c["page"]
    length = [b + n for b, n in zip(s.before, s.q)]
    tables, free, s.n_pages = _tables(s.rng, length, page, spare=5)
    s.max_pages = tables.shape[1]
    s.tables, s.refs = _i32(tables), _zeros(s.n_pages)
    s.free = _zeros(s.n_pages)
    s.free[:len(free)] = _i32(free)
    s.n_free = _i32([len(free)])
    own_at = np.concatenate([b + np.arange(n) for b, n in zip(s.before, s.q)])
    seq = np.repeat(np.arange(c["nseq"]), s.q)
    s.slots = _i32(tables[seq, own_at // page] * page + own_at % page)
    # drafted tokens, and choices that agree with one of a node's children in two of three nodes
    tokens = s.rng.integers(0, 151936, s.t)
    ids = s.rng.integers(0, 151936, s.t)
    for r in range(s.t):
        at = s.starts[seq[r]] + s.parents[r]
        if s.parents[r] >= 0 and s.rng.random() < 0.5:
            ids[at] = tokens[r]
    s.tokens, s.ids = _i32(tokens), _i32(ids)
    s.n_path, s.last, s.keep, s.len_out = (_zeros(c["nseq"]) for _ in range(4))
    s.chosen, s.runs, s.cuts, s.n_free_out = _zeros(c["nseq"], c["path"]), _zeros(c["nseq"], c["path"], 3), _zeros(c["nseq"], 3), _zeros(1)
    _caches(s, c, seed)


def _prepare_fork(s, c, seed):
    page, beams = c["page"], c["beams"]
    s.rng = np.random.default_rng(int(seed))
    prompt, length = _beams(c)
    s.nseq = len(length)
    # beams share their prompt's full pages; all else is their own
    need = [p // page for p in prompt] + [_cdiv(n, page) - prompt[i // beams] // page for i, n in enumerate(length)]
    s.n_pages = sum(need) + s.nseq + 9
    order = s.rng.permutation(s.n_pages).astype(np.int32)
    at = np.concatenate([[0], np.cumsum(need)])
    s.max_pages = max(_cdiv(n, page) for n in length) + 1
    tables, refs = np.zeros((s.nseq, s.max_pages), dtype=np.int32), np.zeros(s.n_pages, dtype=np.int32)
    for i in range(s.nseq):
        r = i // beams
        row = np.concatenate([order[at[r]:at[r + 1]], order[at[c["requests"] + i]:at[c["requests"] + i + 1]]])
        tables[i, :len(row)] = row
    for r in range(c["requests"]):
        refs[order[at[r]:at[r + 1]]] = beams - 1
    free = order[at[-1]:]
    s.tables, s.refs, s.len, s.n_free, s.free = _i32(tables), _i32(refs), _i32(length), _i32([len(free)]), _zeros(s.n_pages)
    s.free[:len(free)] = _i32(free)
    # each beam goes on from one of its request's, the likelier ones more often
    s.src = _i32([i // beams * beams + int(beams * s.rng.random() ** 1.5) for i in range(s.nseq)])
    s.runs = _zeros(s.nseq, 3)
    _caches(s, c, seed)


def _prepare_logp(s, c, seed):
    rows, n, m, k = c["rows"], c["n"], c["m"], c["k"]
    s.x = 3.0 * _randn(seed, 1, rows, n)
    if c["mask"]:  # a grammar's: some rows allow a few tokens, the others most
        few = (torch.arange(rows, device=DEV) % 2 == 0).view(-1, 1)
        s.x.masked_fill_(torch.rand(rows, n, device=DEV, generator=_gen(seed, 2)) > torch.where(few, 0.01, 0.9), -math.inf)
        s.x[:, 0] = 1.0
    s.ids = torch.randint(0, n, (rows, m), device=DEV, generator=_gen(seed, 3), dtype=torch.int32)
    s.logp, s.rank, s.entropy = _zeros(rows, m, dtype=torch.float32), _zeros(rows, m), _zeros(rows, dtype=torch.float32)
    s.top_ids, s.top_logp = _zeros(rows, k), _zeros(rows, k, dtype=torch.float32)


# ---- one pass ----
def run(s):
    kind = s.c["kind"]
    if own:
        return {"plan": _own_plan, "attn": _own_attn, "keep": _own_keep, "fork": _own_fork, "logp": _own_logp}[kind](_hip(), s, s.c)
    return {"plan": _plain_plan, "attn": _plain_attn, "keep": _plain_keep, "fork": _plain_fork, "logp": _plain_logp}[kind](s, s.c)


def _p(t):
    return t.data_ptr() if t is not None and t.numel() else 0


def _padded(s, v, fill):
    """Rows' values as one line of max(q) a sequence."""
    q = s.q_start.long()
    n = int(max(s.q))
    row = q[:-1].view(-1, 1) + torch.arange(n, device=DEV)
    live = row < q[1:].view(-1, 1)
    return torch.where(live, v.long()[row.clamp(max=s.t - 1)], fill), row, live


def _ancestors(parent):
    """[B, Q, Q]: whether j is i or above it; parent: [B, Q]."""
    j = torch.arange(parent.shape[1], device=DEV)
    up = (parent.unsqueeze(2) == j).float() + torch.eye(parent.shape[1], device=DEV)
    return torch.linalg.matrix_power(up, 64) > 0


def _own_plan(hip, s, c):
    hip.tree_step(c["nseq"], _p(s.q_start), _p(s.parent), _p(s.len), s.t, c["words"], _p(s.pos), _p(s.mask), prefix_len=_p(s.prefix_len))
    return s.pos, s.mask


def _plain_plan(s, c):
    parent, row, live = _padded(s, s.parent, -1)
    up = _ancestors(parent)
    depth = up.sum(2) - 1
    pos = s.prefix_len + (s.len - (s.q_start[1:] - s.q_start[:-1])).view(-1, 1) + depth
    s.pos[row[live]] = pos[live].to(torch.int32)
    bits = torch.zeros(*parent.shape, 32 * c["words"], device=DEV, dtype=torch.int64)
    bits[:, :, :parent.shape[1]] = up.long()
    w = (bits.view(*parent.shape, c["words"], 32) << torch.arange(32, device=DEV)).sum(3)
    s.mask[row[live]] = torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)[live]
    return s.pos, s.mask


def _own_attn(hip, s, c):
    P = c["prefix"]
    hip.attn_paged_tree(_p(s.x), _p(s.kc), _p(s.vc), _p(s.gate), _p(s.out), s.t, s.max_q, _p(s.pos), _p(s.q_start), _p(s.len), c["nseq"],
                        _p(s.tables), s.max_pages, c["page"], s.n_pages, c["nh"], c["nkv"], c["hd"], 1.0 / math.sqrt(c["hd"]), _p(s.mask),
                        c["words"], prefix=_p(s.prefix) if P else 0, prefix_len=_p(s.prefix_len) if P else 0, max_prefix=P, sink=_p(s.sink),
                        win=c["win"])
    return s.out


def _plain_attn(s, c):
    nh, nkv, hd, P, page, W = c["nh"], c["nkv"], c["hd"], c["prefix"], c["page"], c["words"]
    G, B, Q = nh // nkv, c["nseq"], s.max_q
    pool_k, pool_v = s.kc.view(-1, page, nkv, hd), s.vc.view(-1, page, nkv, hd)
    pos, row, live = _padded(s, s.pos, 0)
    row = row.clamp(max=s.t - 1)
    q = s.x[row].view(B, Q, nkv, G, hd).permute(0, 2, 1, 3, 4).reshape(B, nkv, Q * G, hd) * (1.0 / math.sqrt(hd))
    k, v = (p[s.tables.long()].view(B, -1, nkv, hd).permute(0, 2, 1, 3).float().contiguous() for p in (pool_k, pool_v))
    L = k.shape[2]
    j = torch.arange(L, device=DEV).view(1, 1, -1)
    base = (s.len - (s.q_start[1:] - s.q_start[:-1])).long().view(B, 1, 1)
    node = (j - base).clamp(0, 32 * W - 1)  # which of the step's rows a key is
    words = s.mask[row].long()  # [B, Q, W]
    bit = (torch.gather(words, 2, (node // 32).expand(B, Q, L)) >> (node % 32)) & 1
    see = (j < s.len.view(B, 1, 1)) & ((j < base) | (bit != 0))
    if c["win"]:
        see = see & ((j >= base) | (j + P > pos.view(B, Q, 1) - c["win"]))
    sc = (q @ k.transpose(2, 3)).view(B, nkv, Q, G, L).masked_fill_(~see.view(B, 1, Q, 1, L), -math.inf)
    if P:
        kp, vp = (p[s.prefix.long()].view(-1, nkv, hd)[:P].transpose(0, 1).float().contiguous() for p in (pool_k, pool_v))
        sp = (q.transpose(0, 1).reshape(nkv, B * Q * G, hd) @ kp.transpose(1, 2)).view(nkv, B, Q, G, P).transpose(0, 1)
        if c["win"]:
            sp = sp.masked_fill((torch.arange(P, device=DEV).view(1, 1, -1) <= pos.view(B, Q, 1) - c["win"]).view(B, 1, Q, 1, P), -math.inf)
        sc = torch.cat([sp, sc], 4)
    m = sc.amax(4, keepdim=True)
    if s.sink is not None:
        sink = s.sink.view(1, nkv, 1, G, 1)
        m = torch.maximum(m, sink)
    m = torch.where(m == -math.inf, 0.0, m)
    e = torch.exp(sc - m)
    den = e.sum(4, keepdim=True)
    if s.sink is not None:
        den = den + torch.exp(sink - m)
    o = e[..., P:].reshape(B, nkv, Q * G, L) @ v
    if P:
        o = o + (e[..., :P].transpose(0, 1).reshape(nkv, B * Q * G, P) @ vp).view(nkv, B, Q * G, hd).transpose(0, 1)
    o = o.view(B, nkv, Q, G, hd) / den
    s.out[row[live]] = o.permute(0, 2, 1, 3, 4).reshape(B, Q, nh, hd)[live]
    if s.gate is not None:
        s.out.mul_(1.0 / (1.0 + torch.exp(-s.gate[:, :, 1])))
    return s.out


def _own_keep(hip, s, c):
    n = c["nseq"]
    hip.tree_accept(n, _p(s.q_start), _p(s.parent), _p(s.tokens), _p(s.ids), _p(s.len), _p(s.slots), s.t, c["words"], c["path"], _p(s.n_path),
                    _p(s.chosen), _p(s.last), _p(s.keep), _p(s.runs))
    hip.kv_rows_move(_p(s.addresses), c["caches"], 2 * s.width, s.n_slots, _p(s.runs), n, c["path"])
    hip.kv_pages_fork(n, 0, _p(s.keep), _p(s.len), _p(s.tables), s.max_pages, c["page"], _p(s.free), s.n_pages, _p(s.n_free), _p(s.refs),
                      _p(s.len_out), _p(s.n_free_out), _p(s.cuts))
    return s.n_path, s.chosen, s.last, s.keep, s.runs, s.kv, s.len_out, s.n_free_out, s.free, s.refs, s.tables


def _plain_keep(s, c):
    page = c["page"]
    parent, row, live = _padded(s, s.parent, -1)
    tokens, slots = _padded(s, s.tokens, -2)[0], _padded(s, s.slots, -1)[0]
    ids = _padded(s, s.ids, -3)[0]
    B, Q = parent.shape
    # a node agrees if the choice after its parent is its token and no sibling before it agrees
    hit = (parent >= 0) & (torch.gather(ids, 1, parent.clamp(min=0)) == tokens)
    j = torch.arange(Q, device=DEV)
    before = hit.unsqueeze(1) & (parent.unsqueeze(1) == parent.unsqueeze(2)) & (j < j.view(-1, 1))
    good = hit & ~before.any(2)
    good[:, 0] = True
    up = _ancestors(parent)
    ok = ~(up & ~good.unsqueeze(1)).any(2) & up[:, :, 0] & live
    place = torch.cumsum(ok, 1) - 1  # where on the path
    ok = ok & (place < c["path"])
    s.n_path.copy_(ok.sum(1))
    seq, node = ok.nonzero(as_tuple=True)
    at = place[seq, node]
    s.chosen.fill_(-1)
    s.chosen[seq, at] = ids[seq, node].to(torch.int32)
    s.last.copy_(s.q_start[:-1] + torch.where(ok, j, -1).amax(1))
    base = s.len - (s.q_start[1:] - s.q_start[:-1])
    s.keep.copy_(base + s.n_path)
    moved = (node != at).long()
    s.runs.zero_()
    src, dst = slots[seq, node], slots[seq, at]
    s.runs[seq, at] = (torch.stack([src, dst, torch.ones_like(src)], 1) * moved.view(-1, 1)).to(torch.int32)
    s.kv[:, dst] = s.kv[:, src]
    # the pages behind
    have, left = (s.len.long() + page - 1) // page, (s.keep.long() + page - 1) // page
    p = torch.arange(s.max_pages, device=DEV)
    back = s.tables.long()[(p >= left.view(-1, 1)) & (p < have.view(-1, 1))]
    top = int(s.n_free)
    s.free[top:top + len(back)] = back.to(torch.int32)
    s.n_free_out.fill_(top + len(back))
    s.len_out.copy_(s.keep)
    return s.n_path, s.chosen, s.last, s.keep, s.runs, s.kv, s.len_out, s.n_free_out, s.free, s.refs, s.tables


def _own_fork(hip, s, c):
    hip.kv_pages_fork(s.nseq, _p(s.src), 0, _p(s.len), _p(s.tables), s.max_pages, c["page"], _p(s.free), s.n_pages, _p(s.n_free), _p(s.refs),
                      _p(s.len), _p(s.n_free), _p(s.runs))
    hip.kv_rows_move(_p(s.addresses), c["caches"], 2 * s.width, s.n_slots, _p(s.runs), s.nseq, 1)
    return s.tables, s.refs, s.len, s.n_free, s.free, s.runs, s.kv


def _plain_fork(s, c):
    page, B = c["page"], s.nseq
    src, old, length, tables = s.src.long(), s.len.long(), s.len.long()[s.src.long()], s.tables.long()
    me, p = torch.arange(B, device=DEV), torch.arange(s.max_pages, device=DEV)
    changed = src != me
    full, rem = length // page, length % page
    # who takes over a sequence's last page: itself, or else the first that goes on from it
    heir = torch.full((B,), B, device=DEV).scatter_reduce(0, src, torch.where(changed, me, -1), "amin")
    heir = torch.where(src[me] == me, me, heir)
    rows = tables[src]
    last = rows[me, full.clamp(max=s.max_pages - 1)]
    takes = (heir[src] == me) & (s.refs.long()[last] == 0)
    need = changed & (rem > 0) & ~takes
    top = int(s.n_free) - 1
    fresh = s.free.long()[top - (torch.cumsum(need, 0) - need.long())]
    held = p < _cdiv_t(old, page).view(-1, 1)
    more = (p < (full + ((rem > 0) & takes)).view(-1, 1)) & changed.view(-1, 1)
    back = held & changed.view(-1, 1)
    refs = s.refs.long()
    refs = refs + torch.bincount(rows[more], minlength=s.n_pages) - torch.bincount(tables[back], minlength=s.n_pages)
    # pages that nobody holds, where they are first met
    flat = (me.view(-1, 1) * s.max_pages + p)[back]
    page_of = tables[back]
    first = torch.full((s.n_pages,), 1 << 40, device=DEV).scatter_reduce(0, page_of, flat, "amin")
    gone = page_of[(refs[page_of] < 0) & (first[page_of] == flat)]
    new = torch.where(more, rows, tables)
    cell = need.view(-1, 1) & (p == full.view(-1, 1))
    s.tables.copy_(torch.where(cell, fresh.view(-1, 1), new))
    s.refs.copy_(refs.clamp(min=0))
    s.len.copy_(length)
    top = top + 1 - int(need.sum())
    s.free[top:top + len(gone)] = gone.to(torch.int32)
    s.n_free.fill_(top + len(gone))
    s.runs.copy_(torch.stack([last * page, fresh * page, rem], 1) * need.long().view(-1, 1))
    i = torch.arange(page, device=DEV)
    live = need.view(-1, 1) & (i < rem.view(-1, 1))
    s.kv[:, (fresh.view(-1, 1) * page + i)[live]] = s.kv[:, (last.view(-1, 1) * page + i)[live]]
    return s.tables, s.refs, s.len, s.n_free, s.free, s.runs, s.kv


def _cdiv_t(a, b):
    return (a + b - 1) // b


def _own_logp(hip, s, c):
    hip.logits_logprobs(_p(s.x), c["n"], c["n"], c["rows"], ids=_p(s.ids), m=c["m"], logp=_p(s.logp), rank=_p(s.rank), entropy=_p(s.entropy),
                        k=c["k"], top_ids=_p(s.top_ids), top_logp=_p(s.top_logp))
    return s.logp, s.rank, s.entropy, s.top_ids, s.top_logp


def _plain_logp(s, c):
    y = s.x - s.x.amax(1, keepdim=True)
    e = torch.exp(y)
    total = e.sum(1, keepdim=True)
    ls = torch.log(total)
    ids = s.ids.long()
    s.logp.copy_(torch.gather(y, 1, ids) - ls)
    at = torch.gather(s.x, 1, ids)
    v = torch.arange(c["n"], device=DEV)
    s.rank.copy_(torch.stack([((s.x > at[:, i:i + 1]) | ((s.x == at[:, i:i + 1]) & (v < ids[:, i:i + 1]))).sum(1) + 1 for i in range(c["m"])], 1) if c["m"] else s.rank)
    s.entropy.copy_((ls - torch.where(e > 0, e * y, 0.0).sum(1, keepdim=True) / total).view(-1))
    where = torch.sort(s.x, dim=1, descending=True, stable=True)[1][:, :c["k"]]
    s.top_ids.copy_(where)
    s.top_logp.copy_(torch.gather(y, 1, where) - ls)
    return s.logp, s.rank, s.entropy, s.top_ids, s.top_logp


# ---- what a pass cannot do without ----
def work(case):
    c, kind = case, case["kind"]
    if kind == "logp":
        return {"bytes": 4 * c["rows"] * c["n"] + c["rows"] * (12 * c["m"] + 8 * c["k"] + 4), "flops": c["rows"] * c["n"] * 5}
    if kind == "fork":
        _, length = _beams(c)
        rem = sum(n % c["page"] for n in length) / 2  # about half of the beams go on from another's and copy
        return {"bytes": int(rem * 4 * c["nkv"] * c["hd"] * c["caches"] + sum(8 * _cdiv(n, c["page"]) for n in length)), "flops": 8 * len(length)}
    q, before = _sizes(c)
    if kind == "plan":
        return {"bytes": sum(q) * (8 + 4 * c["words"]) + 8 * c["nseq"], "flops": sum(q) * 8}
    if kind == "keep":
        moved = sum(min(c["path"] - 1, n - 1, 2) for n in q)  # paths are a few nodes long
        return {"bytes": moved * 4 * c["nkv"] * c["hd"] * c["caches"] + sum(q) * 16 + c["nseq"] * (24 + 12 * c["path"]), "flops": sum(q) * 4}
    P, win, nh, nkv, hd = c["prefix"], c["win"] or 1 << 60, c["nh"], c["nkv"], c["hd"]
    depth = [1 + math.log2(n) for n in q]
    keys = sum(n * (min(P + b, win) + d) for n, b, d in zip(q, before, depth))
    own_keys = sum(min(b, win) + n for n, b in zip(q, before))
    first = max(0, min(P + b for b in before) + 1 - win)
    return {"bytes": int(4 * nkv * hd * (max(0, P - first) + own_keys) + (12 if c["gate"] else 8) * sum(q) * nh * hd), "flops": int(4 * hd * nh * keys)}


# ---- the same in 64 bits, plainly ----
def exact(case, seed):
    return {"plan": _exact_plan, "attn": _exact_attn, "keep": _exact_keep, "fork": _exact_fork, "logp": _exact_logp}[case["kind"]](case, seed)


def _exact_plan(c, seed):
    s = prepare(c, seed)
    before = np.repeat(s.before, s.q)
    return (int(s.prefix_len[0]) + before + _depths(s.parents, s.starts)).astype(np.int32), _masks(s.parents, s.starts, c["words"])


def _exact_attn(c, seed):
    s = prepare(c, seed)
    nh, nkv, hd, P, page = c["nh"], c["nkv"], c["hd"], c["prefix"], c["page"]
    out = torch.zeros_like(s.x, dtype=torch.float64)
    depth = torch.from_numpy(_depths(s.parents, s.starts)).to(DEV)

    def rows(pool, table, n):
        return pool.view(-1, page, nkv, hd)[table[:_cdiv(n, page)].long()].view(-1, nkv, hd)[:n].double().transpose(0, 1)

    pre = [rows(p, s.prefix, P) for p in (s.kc, s.vc)]
    for b in range(c["nseq"]):
        at, n, first = int(s.starts[b]), s.q[b], s.before[b]
        key, val = (torch.cat([p, rows(pool, s.tables[b], first + n)], 1) for p, pool in zip(pre, (s.kc, s.vc)))
        above = np.zeros((n, n), dtype=bool)
        for i in range(n):
            if i:
                above[i] = above[s.parents[at + i]]
            above[i, i] = True
        where = P + first + depth[at:at + n].view(-1, 1)
        k = torch.arange(P + first, device=DEV).view(1, -1)
        ok = torch.cat([k > where - (c["win"] or 1 << 40), torch.from_numpy(above).to(DEV)], 1)
        for g in range(nkv):
            h = slice(g * nh // nkv, (g + 1) * nh // nkv)
            sc = torch.where(ok.unsqueeze(1), s.x[at:at + n, h].double() @ key[g].T / math.sqrt(hd), -math.inf)
            if s.sink is not None:
                sc = torch.cat([sc, s.sink[h].double().view(1, -1, 1).expand(n, -1, 1)], 2)
            out[at:at + n, h] = torch.softmax(sc, 2)[:, :, :P + first + n] @ val[g]
    return out if s.gate is None else out * torch.sigmoid(s.gate[:, :, 1].double())


def _exact_keep(c, seed):
    s = prepare(c, seed)
    B, page = c["nseq"], c["page"]
    tokens, ids, slots, tables = (a.cpu().numpy() for a in (s.tokens, s.ids, s.slots, s.tables))
    n_path, last, keep = (np.zeros(B, dtype=np.int32) for _ in range(3))
    chosen, runs = np.full((B, c["path"]), -1, dtype=np.int32), np.zeros((B, c["path"], 3), dtype=np.int32)
    free, top, moves = s.free.cpu().numpy(), int(s.n_free[0]), []
    for b in range(B):
        at, n, path = int(s.starts[b]), s.q[b], [0]
        while len(path) < c["path"]:
            kids = [i for i in range(n) if s.parents[at + i] == path[-1] and tokens[at + i] == ids[at + path[-1]]]
            if not kids:
                break
            path.append(kids[0])
        for i, r in enumerate(path):
            chosen[b, i] = ids[at + r]
            if r != i:
                runs[b, i] = slots[at + r], slots[at + i], 1
                moves.append((slots[at + r], slots[at + i]))
        n_path[b], last[b], keep[b] = len(path), at + path[-1], s.before[b] + len(path)
        for j in range(_cdiv(int(keep[b]), page), _cdiv(s.before[b] + n, page)):
            free[top] = tables[b, j]
            top += 1
    kv = s.kv.clone()
    for a, b in moves:
        kv[:, b] = kv[:, a]
    return n_path, chosen, last, keep, runs, kv, keep, np.array([top], dtype=np.int32), free, s.refs, tables


def _exact_fork(c, seed):
    s = prepare(c, seed)
    page = c["page"]
    src, length, old, refs = (a.cpu().numpy() for a in (s.src, s.len, s.tables, s.refs))
    tables, stack, count, kv = old.copy(), s.free.cpu().numpy(), refs.astype(np.int64), s.kv.clone()
    top, runs, taken = int(s.n_free[0]), np.zeros((s.nseq, 3), dtype=np.int32), set(u for u in range(s.nseq) if src[u] == u)
    for i in range(s.nseq):
        u, n = src[i], int(length[src[i]])
        if u == i:
            continue
        j, rem = n // page, n % page
        tables[i, :j] = old[u, :j]
        for p in old[u, :j]:
            count[p] += 1
        if rem:
            heir = u not in taken
            taken.add(u)
            if heir and refs[old[u, j]] == 0:
                tables[i, j] = old[u, j]
                count[old[u, j]] += 1
            else:
                top -= 1
                tables[i, j] = stack[top]
                runs[i] = old[u, j] * page, stack[top] * page, rem
                kv[:, stack[top] * page:stack[top] * page + rem] = s.kv[:, old[u, j] * page:old[u, j] * page + rem]
    back = [p for i in range(s.nseq) if src[i] != i for p in old[i, :_cdiv(int(length[i]), page)]]
    for p in back:
        count[p] -= 1
    for p in back:
        if count[p] < 0:
            count[p] = 0
            stack[top] = p
            top += 1
    return tables, count.astype(np.int32), length[src], np.array([top], dtype=np.int32), stack, runs, kv


def _exact_logp(c, seed):
    s = prepare(c, seed)
    rows, m, k = c["rows"], c["m"], c["k"]
    logp, rank = torch.zeros(rows, m, dtype=torch.float64, device=DEV), torch.zeros(rows, m, dtype=torch.int32, device=DEV)
    entropy, top_ids, top_logp = torch.zeros(rows, dtype=torch.float64, device=DEV), torch.zeros(rows, k, dtype=torch.int32, device=DEV), torch.zeros(rows, k, dtype=torch.float64, device=DEV)
    for r in range(rows):
        y = torch.log_softmax(s.x[r].double(), 0)
        p = torch.exp(y)
        entropy[r] = -(p * torch.where(p > 0, y, 0.0)).sum()
        order = torch.argsort(s.x[r], descending=True, stable=True)
        place = torch.empty_like(order)
        place[order] = torch.arange(c["n"], device=DEV)
        logp[r], rank[r] = y[s.ids[r].long()], (place[s.ids[r].long()] + 1).to(torch.int32)
        top_ids[r], top_logp[r] = order[:k].to(torch.int32), y[order[:k]]
    return logp, rank, entropy, top_ids, top_logp
