"""The operators that serve a batch of sequences over a paged f16 KV cache, as workloads that are timed and checked.

Kinds of case, and what they stand for:
  pages   `kv_pages_step`: one step's block tables, slot map and positions from the sequences' lengths and new tokens
          (sequences that end give their pages back first)
  rope    `rms_norm_rope_qk_paged`: a layer's q/k head norms and rotation at each token's own position, keys and values
          stored into the pages, heads read in place from the fused q/k/v rows
  attn    `attn_paged`: attention of a ragged batch (one token a sequence, a few speculative ones, or prompt chunks) over
          the pages, with or without a prefix that all of the batch shares
  logits  `logits_process`: penalties for repeated tokens, biases and grammar masks on a step's logits, and the greedy
          choice

`own` false computes them plainly in torch, true through the backend. Sequence lengths follow from a case's values alone;
the data, and where pages lie, from the seed.
"""
import math
import random

import numpy as np
import torch

own = False
DEV = "cuda"
EPS = 1e-6
BASE = 1e6
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
        # a step of a few decoding sequences: nothing but latency
        {"name": "pages_decode_8", "kind": "pages", "nseq": 8, "page": 64, "max_len": 4096, "tokens": 8, "ends": 0, "mix": 1},
        # a busy server's step: hundreds decode, some end, some bring prompts
        {"name": "pages_mixed_512", "kind": "pages", "nseq": 512, "page": 16, "max_len": 8192, "tokens": 8192, "ends": 20, "mix": 2},
        # a layer of a decode step
        {"name": "rope_decode_32", "kind": "rope", "t": 32, "nh": 32, "nkv": 4, "hd": 128, "n_rot": 128, "page": 16, "mix": 3},
        # a layer of a full prefill chunk made of several prompts
        {"name": "rope_chunk_4096", "kind": "rope", "t": 4096, "nh": 32, "nkv": 4, "hd": 128, "n_rot": 128, "page": 64, "mix": 4},
        # one sequence of a chat turn's length
        {"name": "attn_1_short", "kind": "attn", "nseq": 1, "max_q": 1, "q": 0, "min_len": 500, "max_len": 600, "prefix": 0, "page": 64, "nh": 32, "nkv": 4, "hd": 128, "win": 0, "sink": 0, "gate": 0, "mix": 5},
        # decode of a batch with contexts of very different lengths
        {"name": "attn_64_ragged", "kind": "attn", "nseq": 64, "max_q": 1, "q": 0, "min_len": 100, "max_len": 24000, "prefix": 0, "page": 16, "nh": 32, "nkv": 4, "hd": 128, "win": 0, "sink": 0, "gate": 0, "mix": 6},
        # decode of a batch that shares a long system prompt or document
        {"name": "attn_prefix_64", "kind": "attn", "nseq": 64, "max_q": 1, "q": 0, "min_len": 1, "max_len": 1000, "prefix": 16000, "page": 64, "nh": 32, "nkv": 4, "hd": 128, "win": 0, "sink": 0, "gate": 0, "mix": 7},
        # speculative tokens over a shared prefix, small heads, sink logits and output gates
        {"name": "attn_spec_24", "kind": "attn", "nseq": 24, "max_q": 4, "q": 0, "min_len": 4, "max_len": 700, "prefix": 6001, "page": 32, "nh": 16, "nkv": 8, "hd": 64, "win": 0, "sink": 1, "gate": 1, "mix": 8},
        # prompt chunks of several sequences, some from their start and some with earlier context, among decoding ones
        {"name": "attn_chunks_2501", "kind": "attn", "nseq": 10, "max_q": 1100, "q": 2501, "min_len": 500, "max_len": 6000, "prefix": 0, "page": 64, "nh": 32, "nkv": 4, "hd": 128, "win": 0, "sink": 0, "gate": 0, "mix": 9},
        # the choice of one sequence's next token
        {"name": "logits_1", "kind": "logits", "rows": 1, "n": 151936, "hist": 1000, "last": 0, "bias": 0, "mask": 0, "mix": 10},
        # a grammar over a few sequences, an odd vocabulary
        {"name": "logits_grammar_8", "kind": "logits", "rows": 8, "n": 32003, "hist": 300, "last": 64, "bias": 20, "mask": 1, "mix": 11},
        # a full batch with long histories
        {"name": "logits_64", "kind": "logits", "rows": 64, "n": 151936, "hist": 4096, "last": 0, "bias": 100, "mask": 1, "mix": 12},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["pages", "rope", "attn", "attn", "attn", "logits", "logits"])
    mix, page = rng.randrange(1 << 20), rng.choice([16, 32, 64, 128])
    if kind == "pages":
        nseq = _log(rng, 1, 512)
        return {"kind": kind, "nseq": nseq, "page": page, "max_len": _log(rng, 256, 8192), "tokens": max(nseq, _log(rng, 1, 8192)), "ends": rng.randrange(nseq // 8 + 1), "mix": mix}
    if kind == "logits":
        return {"kind": kind, "rows": _log(rng, 1, 64), "n": rng.choice([_log(rng, 1000, 151936), 151936]), "hist": _log(rng, 1, 4096), "last": rng.choice([0, 0, 64, 256]), "bias": rng.choice([0, 1, 300]), "mask": rng.choice([0, 1]), "mix": mix}
    nh, nkv, hd = rng.choice([(32, 4, 128), (32, 4, 128), (32, 8, 128), (16, 8, 64), (16, 16, 128), (16, 2, 64)])
    if kind == "rope":
        return {"kind": kind, "t": _log(rng, 1, 4096), "nh": nh, "nkv": nkv, "hd": hd, "n_rot": rng.choice([hd, hd, hd // 2]), "page": page, "mix": mix}
    c = {"kind": kind, "page": page, "nh": nh, "nkv": nkv, "hd": hd, "win": rng.choice([0, 0, 0, 1024]), "sink": rng.choice([0, 0, 1]), "gate": rng.choice([0, 0, 1]), "mix": mix}
    form = rng.choice(["one", "one", "shared", "shared", "spec", "chunks"])
    c["prefix"] = _log(rng, 100, 16000) if form == "shared" else rng.choice([0, _log(rng, 100, 2000)])
    if form == "chunks":
        c |= {"nseq": _log(rng, 1, 12), "max_q": 700, "q": _log(rng, 30, 1500), "min_len": 1, "max_len": _log(rng, 100, 3000)}
    else:
        c |= {"nseq": _log(rng, 1, 64), "max_q": rng.randrange(2, 9) if form == "spec" else 1, "q": 0, "min_len": 1, "max_len": _log(rng, 60, 1000 if form == "shared" else 8000)}
    return c


# ---- lengths: what a case's values alone say ----
def _lens(c):
    """(new tokens, cached tokens with the new ones) of each sequence of an attention case."""
    r = random.Random(c["mix"])
    length = [_log(r, c["min_len"], c["max_len"]) for _ in range(c["nseq"])]
    q = [r.randint(1, c["max_q"]) if c["max_q"] < 16 else 1 for _ in range(c["nseq"])]
    left = c["q"]  # prompt chunks: the first sequences share c["q"] tokens, the others decode
    for i in range(c["nseq"] if left else 0):
        if left <= 0:
            break
        q[i] = min(left, c["max_q"], max(1, int(left * r.uniform(0.3, 0.9))))
        left -= q[i]
        if i % 2 == 0:
            length[i] = 0  # a prompt from its start
    return q, [n + k for k, n in zip(q, length)]


def _steps(c):
    """(new tokens or -1, cached tokens) of each sequence of a page step."""
    r = random.Random(c["mix"])
    length = [_log(r, 1, c["max_len"] - c["tokens"] if c["tokens"] < c["max_len"] // 2 else c["max_len"] // 2) for _ in range(c["nseq"])]
    add = [1] * c["nseq"]
    left = c["tokens"] - c["nseq"]
    while left > 0:
        i, k = r.randrange(c["nseq"]), min(left, r.randint(1, 2048))
        add[i] += k
        left -= k
    for i in r.sample(range(c["nseq"]), c["ends"]):
        add[i] = -1
    return add, length


# ---- inputs ----
def _gen(seed, part):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1009 + part) % (1 << 62))
    return g


def _randn(seed, part, *shape):
    return torch.randn(*shape, device=DEV, dtype=torch.float32, generator=_gen(seed, part))


def _i32(v):
    return torch.tensor(np.asarray(v), device=DEV, dtype=torch.int32)


def _zeros(*shape, dtype=torch.float32):
    return torch.zeros(*shape, device=DEV, dtype=dtype)


def _cdiv(a, b):
    return -(-a // b)


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
    s, c = _State(), case
    s.c = c
    {"pages": _prepare_pages, "rope": _prepare_rope, "attn": _prepare_attn, "logits": _prepare_logits}[c["kind"]](s, c, seed)
    return s


def _prepare_pages(s, c, seed):
    add, length = _steps(c)
    take = [max(a, 0) for a in add]
    page = c["page"]
    want = sum(_cdiv(n + a, page) - _cdiv(n, page) for n, a in zip(length, take))
    tables, free, n_pages = _tables(np.random.default_rng(int(seed)), length, page, spare=want + 8)
    s.max_pages = _cdiv(max(n + a for n, a in zip(length, take)), page)
    s.tables = _zeros(c["nseq"], s.max_pages, dtype=torch.int32)
    s.tables[:, :tables.shape[1]] = torch.from_numpy(tables).to(DEV)
    s.free = _zeros(n_pages + 1, dtype=torch.int32)  # (one spare entry for the plain form's writes that go nowhere)
    s.free[:len(free)] = torch.from_numpy(free).to(DEV)
    s.n_pages, s.t_max = n_pages, sum(take)
    s.add, s.len, s.n_free, s.prefix_len = _i32(add), _i32(length), _i32([len(free)]), _i32([int(seed) % 5000])
    s.q_start, s.pos, s.slots = (_zeros(k, dtype=torch.int32) for k in (c["nseq"] + 1, s.t_max, s.t_max))
    s.len_out, s.n_free_out = _zeros(c["nseq"], dtype=torch.int32), _zeros(1, dtype=torch.int32)


def _prepare_rope(s, c, seed):
    t, nh, nkv, hd, page = c["t"], c["nh"], c["nkv"], c["hd"], c["page"]
    r = random.Random(c["mix"])
    pos = []
    while len(pos) < t:  # sequences of one to many tokens, at positions up to 100000
        k, at = min(t - len(pos), _log(r, 1, 1000) if t > 256 else 1), _log(r, 1, 100000)
        pos += range(at, at + k)
    s.n_slots = _cdiv(t, page) * page + page
    slots = np.random.default_rng(int(seed)).permutation(s.n_slots)[:t].astype(np.int32)
    s.pos, s.slots = _i32(pos), _i32(slots)
    s.qkv = _randn(seed, 1, t, (nh + 2 * nkv) * hd)
    s.qw, s.kw = 1.0 + 0.1 * _randn(seed, 2, hd), 1.0 + 0.1 * _randn(seed, 3, hd)
    s.qo = _zeros(t, nh, hd)
    s.kc, s.vc = (_zeros(s.n_slots, nkv, hd, dtype=torch.float16) for _ in range(2))


def _attn_data(c, seed):
    """q, the page pool, tables, prefix pages, sink logits and gates of an attention case."""
    nh, nkv, hd, page, P = c["nh"], c["nkv"], c["hd"], c["page"], c["prefix"]
    q, length = _lens(c)
    t = sum(q)
    tables, _, n_pages = _tables(np.random.default_rng(int(seed)), length + [P], page)
    d = _State()
    d.t, d.n_pages, d.max_pages = t, n_pages, max(1, max(_cdiv(n, page) for n in length))
    d.prefix = torch.from_numpy(tables[-1, :max(1, _cdiv(P, page))].copy()).to(DEV)
    d.tables = torch.from_numpy(tables[:-1, :d.max_pages].copy()).to(DEV)
    d.q = 1.5 * _randn(seed, 1, t, nh, hd)
    d.kc = _randn(seed, 2, n_pages * page, nkv, hd).to(torch.float16)
    d.vc = (0.5 * _randn(seed, 3, n_pages * page, nkv, hd)).to(torch.float16)
    d.sink = _randn(seed, 4, nh) if c["sink"] else None
    d.gate = _randn(seed, 5, t, nh, 2, hd) if c["gate"] else None
    return d, q, length


def _prepare_attn(s, c, seed):
    d, q, length = _attn_data(c, seed)
    s.d = d
    s.q_start = _i32(np.concatenate([[0], np.cumsum(q)]))
    s.pos = _i32(np.concatenate([c["prefix"] + n - k + np.arange(k) for k, n in zip(q, length)]))
    s.len, s.prefix_len = _i32(length), _i32([c["prefix"]])
    s.max_q = max(q)
    s.out = torch.zeros_like(d.q)


def _logits_data(c, seed):
    rows, n = c["rows"], c["n"]
    rng = np.random.default_rng(int(seed) + 77)
    d = _State()
    d.x = 4.0 * _randn(seed, 1, rows, n)
    # a history repeats itself: tokens of a Zipf law over a permutation of the vocabulary
    rank = (np.minimum(rng.zipf(1.2, size=(rows, c["hist"])), 1 << 40) - 1) % n
    d.hist = _i32((rank * 7919 + np.arange(rows)[:, None] * 131) % n)
    lens = rng.integers(max(1, c["hist"] // 2), c["hist"] + 1, rows)
    d.hist_len, d.hist_from = _i32(lens), _i32(lens // 3)
    d.pen = torch.from_numpy(np.stack([rng.uniform(1.0, 1.5, rows), rng.uniform(0, 0.5, rows), rng.uniform(0, 0.5, rows)], 1).astype(np.float32)).to(DEV)
    per = rng.integers(0, c["bias"] + 1, rows) if c["bias"] else np.zeros(rows, dtype=np.int64)
    d.bias_start = _i32(np.concatenate([[0], np.cumsum(per)]))
    d.n_bias = int(per.sum())
    d.bias_ids = _i32(rng.integers(0, n, max(1, d.n_bias)))
    d.bias_vals = torch.from_numpy(rng.normal(0, 5, max(1, d.n_bias)).astype(np.float32)).to(DEV)
    d.mask = None
    if c["mask"]:  # some rows' grammars allow a few tokens, the others most
        words = _cdiv(n, 32)
        few = torch.from_numpy(rng.random(rows) < 0.5).to(DEV).view(-1, 1)
        bits = torch.rand(rows, words * 32, device=DEV, generator=_gen(seed, 2)) < torch.where(few, 0.001, 0.9)
        bits[:, 0] = True
        w = (bits.view(rows, words, 32).to(torch.int64) << torch.arange(32, device=DEV)).sum(2)
        d.mask = torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)
    return d


def _prepare_logits(s, c, seed):
    s.d = _logits_data(c, seed)
    s.out = torch.zeros_like(s.d.x)
    s.ids = _zeros(c["rows"], dtype=torch.int32)


# ---- one pass ----
def run(s):
    kind = s.c["kind"]
    if own:
        return {"pages": _own_pages, "rope": _own_rope, "attn": _own_attn, "logits": _own_logits}[kind](_hip(), s, s.c)
    return {"pages": _plain_pages, "rope": _plain_rope, "attn": _plain_attn, "logits": _plain_logits}[kind](s, s.c)


def _p(t):
    return t.data_ptr() if t is not None else 0


def _own_pages(hip, s, c):
    hip.kv_pages_step(c["nseq"], _p(s.add), _p(s.len), _p(s.tables), s.max_pages, c["page"], _p(s.free), s.n_pages, _p(s.n_free),
                      s.t_max, _p(s.q_start), _p(s.pos), _p(s.slots), _p(s.len_out), _p(s.n_free_out), prefix_len=_p(s.prefix_len))
    return s.q_start, s.pos, s.slots, s.len_out, s.n_free_out, s.tables, s.free[:s.n_pages]


def _plain_pages(s, c):
    page, n, nseq = c["page"], s.len.long(), c["nseq"]
    end, take = s.add < 0, s.add.clamp(min=0).long()
    ends = torch.cumsum(take, 0)
    starts = ends - take
    j = torch.arange(s.max_pages, device=DEV)
    back = torch.where(end, (n + page - 1) // page, 0)
    at = s.n_free.long() + (torch.cumsum(back, 0) - back).view(-1, 1) + j
    s.free[torch.where(j < back.view(-1, 1), at, s.n_pages).view(-1)] = s.tables.view(-1)
    top = s.n_free.long() + back.sum()
    have = (n + page - 1) // page
    need = (n + take + page - 1) // page - have
    bad = (take > 0) & ((n + take > s.max_pages * page) | (ends > s.t_max))
    need = torch.where(bad, 0, need)
    off = torch.cumsum(need, 0) - need
    bad = bad | ((need > 0) & (off + need > top))
    t = torch.arange(s.t_max, device=DEV)
    seq = torch.searchsorted(ends, t, right=True).clamp(max=nseq - 1)
    i = n[seq] + t - starts[seq]
    pi = i // page
    new = pi >= have[seq]
    from_free = s.free[(top - 1 - (off[seq] + pi - have[seq])).clamp(0, s.n_pages)]
    pages = torch.where(new, from_free, s.tables[seq, pi.clamp(max=s.max_pages - 1)])
    live = (t < ends[-1]) & ~bad[seq]
    s.slots.copy_(torch.where(live, pages * page + i % page, -1))
    s.pos.copy_(torch.where(t < ends[-1], s.prefix_len + i, -1))
    fresh = (live & new & (i % page == 0)).view(-1, 1)
    cell = torch.where(fresh.view(-1), seq * s.max_pages + pi, 0)
    s.tables.view(-1)[cell] = torch.where(fresh.view(-1), pages, s.tables.view(-1)[0]).to(torch.int32)
    s.q_start[0] = 0
    s.q_start[1:] = ends.clamp(max=s.t_max)
    s.len_out.copy_(torch.where(end, 0, torch.where(bad, n, n + take)))
    s.n_free_out.copy_(top - torch.where(bad, 0, need).sum())
    return s.q_start, s.pos, s.slots, s.len_out, s.n_free_out, s.tables, s.free[:s.n_pages]


def _own_rope(hip, s, c):
    nh, nkv, hd = c["nh"], c["nkv"], c["hd"]
    w, q = (nh + 2 * nkv) * hd, _p(s.qkv)
    hip.rms_norm_rope_qk_paged(q, w, hd, _p(s.qw), _p(s.qo), nh, q + 4 * nh * hd, w, _p(s.kw), nkv, hd, EPS, c["n_rot"], _p(s.pos), BASE,
                               q + 4 * (nh + nkv) * hd, w, _p(s.kc), _p(s.vc), _p(s.slots), s.n_slots, c["t"])
    return s.qo, s.kc, s.vc


def _plain_rope(s, c):
    t, nh, nkv, hd, half = c["t"], c["nh"], c["nkv"], c["hd"], c["n_rot"] // 2
    x = s.qkv.view(t, nh + 2 * nkv, hd)
    h, v = x[:, :nh + nkv], x[:, nh + nkv:]
    w = torch.cat([s.qw.expand(nh, hd), s.kw.expand(nkv, hd)])
    y = h / torch.sqrt((h * h).mean(2, keepdim=True) + EPS) * w
    freq = BASE ** (-2.0 * torch.arange(half, device=DEV, dtype=torch.float64) / c["n_rot"])
    a = s.pos.double().view(-1, 1, 1) * freq
    sn, cs = torch.sin(a).float(), torch.cos(a).float()
    p, q = y[:, :, :half], y[:, :, half:2 * half]
    y = torch.cat([p * cs - q * sn, p * sn + q * cs, y[:, :, 2 * half:]], 2)
    s.qo.copy_(y[:, :nh])
    at = s.slots.long()
    s.kc[at] = y[:, nh:].half()
    s.vc[at] = v.half()
    return s.qo, s.kc, s.vc


def _own_attn(hip, s, c):
    d = s.d
    hip.attn_paged(_p(d.q), _p(d.kc), _p(d.vc), _p(d.gate), _p(s.out), d.t, s.max_q, _p(s.pos), _p(s.q_start), _p(s.len),
                   c["nseq"], _p(d.tables), d.max_pages, c["page"], d.n_pages, c["nh"], c["nkv"], c["hd"], 1.0 / math.sqrt(c["hd"]),
                   prefix=_p(d.prefix) if c["prefix"] else 0, prefix_len=_p(s.prefix_len) if c["prefix"] else 0, max_prefix=c["prefix"],
                   sink=_p(d.sink), win=c["win"])
    return s.out


def _plain_attn(s, c):
    d, nh, nkv, hd, P, page = s.d, c["nh"], c["nkv"], c["hd"], c["prefix"], c["page"]
    G, B, Q = nh // nkv, c["nseq"], s.max_q
    pool_k, pool_v = d.kc.view(-1, page, nkv, hd), d.vc.view(-1, page, nkv, hd)
    # queries padded to Q a sequence: [B, nkv, Q G, hd]
    row = s.q_start[:-1].view(-1, 1) + torch.arange(Q, device=DEV)
    live = row < s.q_start[1:].view(-1, 1)
    row = row.clamp(max=d.t - 1)
    pos = s.pos[row]
    q = d.q[row].view(B, Q, nkv, G, hd).permute(0, 2, 1, 3, 4).reshape(B, nkv, Q * G, hd) * (1.0 / math.sqrt(hd))
    # own keys and values: [B, nkv, L, hd]
    k, v = (p[d.tables.long()].view(B, -1, nkv, hd).permute(0, 2, 1, 3).float().contiguous() for p in (pool_k, pool_v))
    L = k.shape[2]
    j = torch.arange(L, device=DEV).view(1, 1, -1)
    at = pos.view(B, Q, 1)
    hide = (j + P > at) | (j >= s.len.view(B, 1, 1))
    if c["win"]:
        hide = hide | (j + P <= at - c["win"])
    sc = (q @ k.transpose(2, 3)).view(B, nkv, Q, G, L).masked_fill_(hide.view(B, 1, Q, 1, L), -math.inf)
    if P:
        kp, vp = (p[d.prefix.long()].view(-1, nkv, hd)[:P].transpose(0, 1).float().contiguous() for p in (pool_k, pool_v))
        qp = q.transpose(0, 1).reshape(nkv, B * Q * G, hd)
        sp = (qp @ kp.transpose(1, 2)).view(nkv, B, Q, G, P).transpose(0, 1)
        if c["win"]:
            sp = sp.masked_fill((torch.arange(P, device=DEV).view(1, 1, -1) <= at - c["win"]).view(B, 1, Q, 1, P), -math.inf)
        sc = torch.cat([sp, sc], 4)
    m = sc.amax(4, keepdim=True)
    if d.sink is not None:
        sink = d.sink.view(1, nkv, 1, G, 1)
        m = torch.maximum(m, sink)
    m = torch.where(m == -math.inf, 0.0, m)
    e = torch.exp(sc - m)
    den = e.sum(4, keepdim=True)
    if d.sink is not None:
        den = den + torch.exp(sink - m)
    o = e[..., P:].reshape(B, nkv, Q * G, L) @ v
    if P:
        o = o + (e[..., :P].transpose(0, 1).reshape(nkv, B * Q * G, P) @ vp).view(nkv, B, Q * G, hd).transpose(0, 1)
    o = o.view(B, nkv, Q, G, hd) / den
    s.out[row[live]] = o.permute(0, 2, 1, 3, 4).reshape(B, Q, nh, hd)[live]
    if d.gate is not None:
        s.out.mul_(1.0 / (1.0 + torch.exp(-d.gate[:, :, 1])))
    return s.out


def _own_logits(hip, s, c):
    d, n = s.d, c["n"]
    hip.logits_process(_p(d.x), n, _p(s.out), n, n, c["rows"], hist=_p(d.hist), hist_stride=c["hist"], hist_len=_p(d.hist_len),
                       hist_from=_p(d.hist_from), last=c["last"], pen=_p(d.pen), bias_start=_p(d.bias_start) if d.n_bias else 0,
                       bias_ids=_p(d.bias_ids), bias_vals=_p(d.bias_vals), n_bias=d.n_bias, mask=_p(d.mask), mask_stride=_cdiv(n, 32),
                       ids=_p(s.ids))
    return s.out, s.ids


def _plain_logits(s, c):
    d, n, rows = s.d, c["n"], c["rows"]
    i = torch.arange(c["hist"], device=DEV)
    end = d.hist_len.view(-1, 1)
    inside = i < end
    if c["last"]:
        inside = inside & (i >= end - c["last"])
    tok = d.hist.long()
    seen = torch.zeros(rows, n + 1, device=DEV, dtype=torch.int32).scatter_add_(1, torch.where(inside, tok, n), torch.ones_like(d.hist))[:, :n] > 0
    late = inside & (i >= d.hist_from.view(-1, 1))
    cnt = torch.zeros(rows, n + 1, device=DEV, dtype=torch.int32).scatter_add_(1, torch.where(late, tok, n), torch.ones_like(d.hist))[:, :n]
    rep, freq, pres = (d.pen[:, k:k + 1] for k in range(3))
    y = torch.where(seen, torch.where(d.x > 0, d.x / rep, d.x * rep), d.x)
    y = y - freq * cnt
    y = torch.where(cnt > 0, y - pres, y)
    if d.n_bias:
        e = torch.arange(d.n_bias, device=DEV)
        r = torch.searchsorted(d.bias_start[1:].long(), e, right=True)
        last = torch.full((rows * n,), -1, device=DEV, dtype=torch.int64).scatter_reduce_(0, r * n + d.bias_ids.long(), e, "amax").view(rows, n)
        y = torch.where(last >= 0, y + d.bias_vals[last.clamp(min=0)], y)
    if d.mask is not None:
        v = torch.arange(n, device=DEV)
        ok = ((d.mask[:, v // 32] >> (v % 32)) & 1) != 0
        y = torch.where(ok, y, -math.inf)
        s.ids.copy_(torch.where(ok.any(1), torch.argmax(y, 1), -1))
    else:
        s.ids.copy_(torch.argmax(y, 1))
    s.out.copy_(y)
    return s.out, s.ids


# ---- what a pass cannot do without ----
def work(case):
    c, kind = case, case["kind"]
    if kind == "pages":
        add, length = _steps(c)
        t = sum(max(a, 0) for a in add)
        pages = sum(_cdiv(n + a, c["page"]) - _cdiv(n, c["page"]) if a >= 0 else _cdiv(n, c["page"]) for n, a in zip(length, add))
        return {"bytes": 16 * c["nseq"] + 8 * t + 8 * pages, "flops": 2 * t + 8 * c["nseq"]}
    if kind == "rope":
        t, nh, nkv, hd = c["t"], c["nh"], c["nkv"], c["hd"]
        return {"bytes": 4 * t * (2 * nh + 3 * nkv) * hd + 8 * t, "flops": 8 * t * (nh + nkv) * hd}
    if kind == "logits":
        return {"bytes": c["rows"] * (8 * c["n"] + (c["n"] // 8 if c["mask"] else 0) + 3 * c["hist"]), "flops": 4 * c["rows"] * c["n"]}
    q, length = _lens(c)
    P, win, nh, nkv, hd = c["prefix"], c["win"] or 1 << 60, c["nh"], c["nkv"], c["hd"]
    keys = sum(min(P + n - k + i + 1, win) for k, n in zip(q, length) for i in range(k))
    own_keys = sum(min(n, win + k - 1) for k, n in zip(q, length))
    first = max(0, min(P + n - k + 1 for k, n in zip(q, length)) - win)  # the first prefix key that any row sees
    return {"bytes": 4 * nkv * hd * (max(0, P - first) + own_keys) + (12 if c["gate"] else 8) * sum(q) * nh * hd, "flops": 4 * hd * nh * keys}


# ---- the same in 64 bits, plainly ----
def exact(case, seed):
    return {"pages": _exact_pages, "rope": _exact_rope, "attn": _exact_attn, "logits": _exact_logits}[case["kind"]](case, seed)


def _exact_pages(c, seed):
    s = prepare(c, seed)
    add, length = _steps(c)
    page, P = c["page"], int(s.prefix_len[0])
    tables, free = s.tables.cpu().numpy().copy(), s.free.cpu().numpy().copy()
    stack = list(free[:int(s.n_free[0])])
    for a, n, row in zip(add, length, tables):
        if a < 0:
            stack += list(row[:_cdiv(n, page)])
    free[:len(stack)] = stack
    q_start, pos, slots, length_out = [0], [], [], []
    for a, n, row in zip(add, length, tables):
        for i in range(n, n + max(a, 0)):
            if i % page == 0:
                row[i // page] = stack.pop()
            pos.append(P + i)
            slots.append(row[i // page] * page + i % page)
        q_start.append(len(pos))
        length_out.append(0 if a < 0 else n + a)
    return tuple(np.asarray(x, dtype=np.int32) for x in (q_start, pos, slots, length_out, [len(stack)], tables, free[:s.n_pages]))


def _exact_rope(c, seed):
    s = prepare(c, seed)
    t, nh, nkv, hd, half = c["t"], c["nh"], c["nkv"], c["hd"], c["n_rot"] // 2
    x = s.qkv.double().view(t, -1, hd)
    angle = s.pos.double().view(-1, 1, 1) * torch.exp(torch.arange(half, device=DEV, dtype=torch.float64) * (-math.log(BASE) / half))
    turn = torch.polar(torch.ones_like(angle), angle)

    def head(h, w):
        h = h * torch.rsqrt(h.square().mean(2, keepdim=True) + EPS) * w.double()
        z = torch.complex(h[..., :half], h[..., half:2 * half]) * turn
        return torch.cat([z.real, z.imag, h[..., 2 * half:]], 2)

    kc, vc = s.kc.double(), s.vc.double()
    kc[s.slots.long()] = head(x[:, nh:nh + nkv], s.kw)
    vc[s.slots.long()] = x[:, nh + nkv:]
    return head(x[:, :nh], s.qw), kc, vc


def _exact_attn(c, seed):
    d, q, length = _attn_data(c, seed)
    nh, nkv, hd, P, page = c["nh"], c["nkv"], c["hd"], c["prefix"], c["page"]
    out = torch.zeros_like(d.q, dtype=torch.float64)

    def rows(pool, table, n):
        return pool.view(-1, page, nkv, hd)[table[:_cdiv(n, page)].long()].view(-1, nkv, hd)[:n].double().transpose(0, 1)

    pre = [rows(p, d.prefix, P) for p in (d.kc, d.vc)]
    at = 0
    for b, (k, n) in enumerate(zip(q, length)):
        key, val = (torch.cat([p, rows(pool, d.tables[b], n)], 1) for p, pool in zip(pre, (d.kc, d.vc)))
        where = P + n - k + torch.arange(k, device=DEV).view(-1, 1)
        seen = torch.arange(P + n, device=DEV).view(1, -1)
        ok = (seen <= where) & (seen > where - (c["win"] or 1 << 40))
        for g in range(nkv):
            h = slice(g * nh // nkv, (g + 1) * nh // nkv)
            sc = torch.where(ok.unsqueeze(1), d.q[at:at + k, h].double() @ key[g].T / math.sqrt(hd), -math.inf)
            if d.sink is not None:
                sc = torch.cat([sc, d.sink[h].double().view(1, -1, 1).expand(k, -1, 1)], 2)
            out[at:at + k, h] = torch.softmax(sc, 2)[:, :, :P + n] @ val[g]
        at += k
    return out if d.gate is None else out * torch.sigmoid(d.gate[:, :, 1].double())


def _exact_logits(c, seed):
    d = _logits_data(c, seed)
    x = d.x.double().cpu().numpy()
    hist, lens, first, pen = (a.cpu().numpy() for a in (d.hist, d.hist_len, d.hist_from, d.pen))
    starts, ids, vals = (a.cpu().numpy() for a in (d.bias_start, d.bias_ids, d.bias_vals))
    for r in range(c["rows"]):
        rep, freq, pres = (float(v) for v in pen[r])
        lo = max(0, int(lens[r]) - c["last"]) if c["last"] else 0
        tok = np.unique(hist[r, lo:lens[r]])
        x[r, tok] = np.where(x[r, tok] > 0, x[r, tok] / rep, x[r, tok] * rep)
        tok, cnt = np.unique(hist[r, max(lo, first[r]):lens[r]], return_counts=True)
        x[r, tok] -= freq * cnt + pres
        for t, b in dict(zip(ids[starts[r]:starts[r + 1]], vals[starts[r]:starts[r + 1]])).items():
            x[r, t] += float(b)
        if d.mask is not None:
            bits = np.unpackbits(d.mask[r].cpu().numpy().view(np.uint8), bitorder="little")[:c["n"]]
            x[r, bits == 0] = -np.inf
    return x, np.argmax(x, 1).astype(np.int32)
