"""The operators for drafted trees and branching sequences together with those of batch serving, as a server runs them: a decode layer
whose steps verify drafted trees gives the tokens that one token a step gives, eager and replayed, through branches, cuts and ends."""
import numpy as np
import pytest

from tests import branch_oracle as B
from tests import serve_oracle as V

from tests.test_gpu_serve import Server, get_i32, i32, up

pytestmark = pytest.mark.gpu
NODES, PATH = 7, 5


class TreeServer(Server):
    """Server whose steps bring a tree of up to NODES tokens a sequence; row 0 of each is the last chosen token."""

    def __init__(self, hip, seed):
        self.rng = np.random.default_rng(seed)
        super().__init__(hip, self.rng)
        self.cache_prefix()
        n, t = self.NSEQ, self.NSEQ * NODES
        self.t, self.slot_rows = t, self.N_PAGES * self.PAGE
        self.parent, self.tokens, self.row_ids, self.mask = (i32(hip, [0] * t) for _ in range(4))
        self.n_path, self.last, self.keep = (i32(hip, [0] * n) for _ in range(3))
        self.chosen, self.runs, self.copies = i32(hip, [0] * n * PATH), i32(hip, [0] * 3 * n * PATH), i32(hip, [0] * 3 * n)
        self.refs, self.src = i32(hip, [0] * self.N_PAGES), i32(hip, [0] * n)
        self.caches = up(hip, np.array([int(self.kc), int(self.vc)], np.uint64))
        self.logp, self.entropy = (up(hip, np.zeros(t, np.float32)) for _ in range(2))
        self.top, self.top_logp = i32(hip, [0] * 3 * t), up(hip, np.zeros(3 * t, np.float32))

    def move(self, runs, per):
        self.hip.kv_rows_move(self.caches, 2, 2 * self.NKV * self.HD, self.slot_rows, runs, self.NSEQ, per)

    def fork(self, src, keep):
        self.hip.kv_pages_fork(self.NSEQ, src, keep, self.len, self.tables, self.MAX_PAGES, self.PAGE, self.free, self.N_PAGES, self.n_free, self.refs, self.len,
                               self.n_free, self.copies, err=self.err)
        self.move(self.copies, 1)

    def step(self):
        """A step of trees: pages, positions and masks, keys and values, attention, choices with their probabilities, the confirmed
        path, its rows where the sequence goes on, the pages behind."""
        hip, n, t = self.hip, self.NSEQ, self.t
        hip.kv_pages_step(n, self.add, self.len, self.tables, self.MAX_PAGES, self.PAGE, self.free, self.N_PAGES, self.n_free, t, self.q_start, self.pos,
                          self.slots, self.len, self.n_free, prefix_len=self.plen, err=self.err)
        hip.tree_step(n, self.q_start, self.parent, self.len, t, 1, self.pos, self.mask, prefix_len=self.plen, err=self.err)
        self.norm_rope(t, self.pos, self.slots)
        hip.attn_paged_tree(self.qo, self.kc, self.vc, 0, self.out, t, NODES, self.pos, self.q_start, self.len, n, self.tables, self.MAX_PAGES, self.PAGE,
                            self.N_PAGES, self.NH, self.NKV, self.HD, self.HD ** -0.5, self.mask, 1, prefix=self.prefix, prefix_len=self.plen,
                            max_prefix=2 * self.PAGE)
        hip.argmax_rows(self.out, self.vocab, t, self.row_ids)
        hip.logits_logprobs(self.out, self.vocab, self.vocab, t, ids=self.row_ids, m=1, logp=self.logp, entropy=self.entropy, k=3, top_ids=self.top,
                            top_logp=self.top_logp)
        hip.tree_accept(n, self.q_start, self.parent, self.tokens, self.row_ids, self.len, self.slots, t, 1, PATH, self.n_path, self.chosen, self.last,
                        self.keep, self.runs)
        self.move(self.runs, PATH)
        self.fork(0, self.keep)

    def check_pool(self):
        """Every page is free or held by as many sequences as refs says."""
        hip, n = self.hip, self.NSEQ
        length, tables, refs = get_i32(hip, self.len, n), get_i32(hip, self.tables, n * self.MAX_PAGES).reshape(n, -1), get_i32(hip, self.refs, self.N_PAGES)
        free = get_i32(hip, self.free, self.N_PAGES - 2)[:get_i32(hip, self.n_free, 1)[0]]
        held = np.bincount(np.concatenate([tables[s, :-(-k // self.PAGE)] for s, k in enumerate(length)] + [free]), minlength=self.N_PAGES)
        np.testing.assert_array_equal(held[:-2], refs[:-2] + 1)
        assert not held[-2:].any()

    def check_cache(self, toks):
        """Each sequence's cached values are its tokens', its keys theirs at their positions (Server.check's bound)."""
        hip, H = self.hip, self.HD
        kc, vc = (hip.get(b, np.float16, self.slot_rows * self.NKV * H).reshape(-1, self.NKV, H) for b in (self.kc, self.vc))
        tables = get_i32(hip, self.tables, self.NSEQ * self.MAX_PAGES).reshape(self.NSEQ, -1)
        assert get_i32(hip, self.len, self.NSEQ).tolist() == [len(x) for x in toks]
        for s, x in enumerate(toks):
            x = np.array(x, np.int64)
            np.testing.assert_array_equal(V.rows_of(vc, tables[s], len(x), self.PAGE)[0], self.tv[x].astype(np.float16))
            k = V.norm_rope(self.tk[x].astype(np.float64), self.kw, 1e-6, H, self.P + np.arange(len(x))[:, None], 1e4)
            pair = np.hypot(k[..., :H // 2], k[..., H // 2:])
            got = V.rows_of(kc, tables[s], len(x), self.PAGE)[0]
            assert (np.abs(got - k) <= 2.0 ** -11 * np.abs(k) + 2.0 ** -15 * np.concatenate([pair, pair], -1) + 2.0 ** -25).all(), s


def plain_tokens(hip, seed, prompts, n):
    """What one token a step chooses after each prompt."""
    sv = Server(hip, np.random.default_rng(seed))
    sv.cache_prefix()
    rows = [len(p) for p in prompts]
    sv.inputs(np.concatenate(prompts))
    hip.htod(np.array(rows, np.int32), sv.add)
    sv.layer(sum(rows), max(rows))
    ids, got = i32(hip, [0] * sv.T), [[] for _ in prompts]
    last = np.cumsum(rows) - 1
    for _ in range(n):
        hip.argmax_rows(sv.out, sv.vocab, sum(rows), ids)
        new = get_i32(hip, ids, sum(rows))[last]
        for s, v in enumerate(new):
            got[s].append(int(v))
        rows, last = [1] * sv.NSEQ, np.arange(sv.NSEQ)
        sv.inputs(new)
        hip.htod(np.array(rows, np.int32), sv.add)
        sv.layer(sv.NSEQ, 1)
    return got


def draft(rng, truth, g, n, vocab):
    """A tree of n tokens below the g-th true one, right ones among them: parents and tokens."""
    parent, tokens, on = [-1], [truth[g - 1]], [0]  # on: true tokens above a node that is on the true line, else None
    for i in range(1, n):
        p = int(rng.integers(0, i)) if rng.random() < 0.4 else i - 1
        right = on[p] is not None and rng.random() < 0.75
        parent.append(p)
        tokens.append(truth[g + on[p]] if right else int(rng.integers(0, vocab)))
        on.append(on[p] + 1 if on[p] is not None and tokens[i] == truth[g + on[p]] else None)
    return parent, tokens


@pytest.mark.parametrize("graph", [False, True])
def test_serving_trees(hip, graph):
    """Steps of trees, waiting sequences, branches and ends between them: the tokens of one a step, the cached rows of the tokens, and
    a whole pool after every step."""
    rng = np.random.default_rng(11)
    sv = TreeServer(hip, 10)
    prompts = [rng.integers(0, sv.vocab, k) for k in (5, 17, 1, 20)]
    truth = plain_tokens(hip, 10, prompts, 60)
    n = sv.NSEQ
    rows = [len(p) for p in prompts]
    sv.inputs(np.concatenate(prompts))
    hip.htod(np.array(rows, np.int32), sv.add)
    sv.layer(sum(rows), max(rows))
    toks, got = [p.tolist() for p in prompts], [[truth[s][0]] for s in range(n)]
    g, paths = None, []
    for k in range(14):
        if k == 5:  # sequence 1 goes on from 0, 2 from 3
            src = [0, 0, 3, 3]
            hip.htod(np.array(src, np.int32), sv.src)
            sv.fork(sv.src, 0)
            toks, got, truth = ([list(v[u]) for u in src] for v in (toks, got, truth))
            sv.check_pool()
            sv.check_cache(toks)
            assert (get_i32(hip, sv.refs, sv.N_PAGES) > 0).any()
        if k == 9:  # 0 ends, and begins again as a cut of 1
            hip.htod(np.array([0] + [96] * (n - 1), np.int32), sv.keep)
            sv.fork(0, sv.keep)
            toks[0], got[0] = [], []
            sv.check_pool()
            sv.check_cache(toks)
            cut = len(toks[1]) - 4
            hip.htod(np.array([1, 1, 2, 3], np.int32), sv.src)
            hip.htod(np.array([cut, 96, 96, 96], np.int32), sv.keep)
            sv.fork(sv.src, sv.keep)
            toks[0], truth[0], got[0] = toks[1][:cut], truth[1], got[1][:cut - len(toks[1])]
            sv.check_pool()
            sv.check_cache(toks)
        sizes = [0 if rng.random() < 0.1 else int(rng.integers(1, NODES + 1)) for _ in range(n)]
        trees = [draft(rng, truth[s], len(got[s]), q, sv.vocab) if q else ([], []) for s, q in enumerate(sizes)]
        parent, tokens = (np.concatenate([np.array(tr[i], np.int64) for tr in trees] + [np.zeros(sv.t, np.int64)])[:sv.t] for i in (0, 1))
        sv.inputs(tokens)
        for v, b in ((sizes, sv.add), (parent, sv.parent), (tokens, sv.tokens)):
            hip.htod(np.asarray(v, np.int32), b)
        if graph and g is None and k == 1:  # (the step before has sized the workspace)
            g = hip.record_graph(sv.step, keep=[sv])
        before = [len(x) for x in toks]
        g.launch() if g else sv.step()
        n_path, chosen = get_i32(hip, sv.n_path, n), get_i32(hip, sv.chosen, n * PATH).reshape(n, PATH)
        q_start = np.concatenate([[0], np.cumsum(sizes)])
        ids = get_i32(hip, sv.row_ids, sv.t)
        want = B.tree_accept(q_start, parent[:q_start[-1]], tokens[:q_start[-1]], ids, np.array(before) + sizes, np.zeros(sv.t, np.int64), 1, PATH)
        np.testing.assert_array_equal(n_path, want["n_path"])
        for s in range(n):
            c = int(n_path[s])
            assert chosen[s, :c].tolist() == truth[s][len(got[s]):len(got[s]) + c] and (chosen[s, c:] == -1).all(), (k, s)
            if c:
                toks[s] = toks[s] + [got[s][-1]] + chosen[s, :c - 1].tolist()
                got[s] = got[s] + chosen[s, :c].tolist()
        paths += n_path[np.array(sizes) > 0].tolist()
        sv.check_pool()
        sv.check_cache(toks)
        # the choices' probabilities from the rows of logits
        m = int(q_start[-1])
        if m:
            x = hip.get(sv.out, np.float32, m * sv.vocab).reshape(m, -1)
            logp, _, h, top, top_logp = B.logprobs(x, ids[:m, None].astype(np.int64), 3)
            np.testing.assert_array_equal(get_i32(hip, sv.top, 3 * m).reshape(m, 3), top)
            assert np.abs(hip.get(sv.logp, np.float32, m) - logp[:, 0]).max() <= 2.0 ** -18 and np.abs(hip.get(sv.entropy, np.float32, m) - h).max() <= 2.0 ** -16
            assert (top[:, 0] == ids[:m]).all()
    assert get_i32(hip, sv.err, 1)[0] == 0 and max(paths) >= 4 and min(paths) == 1
    hip.htod(np.zeros(n, np.int32), sv.keep)
    sv.fork(0, sv.keep)
    assert get_i32(hip, sv.n_free, 1)[0] == sv.n_free0 and not get_i32(hip, sv.refs, sv.N_PAGES).any()
    if g:
        g.close()


class PartsServer(TreeServer):
    """TreeServer whose step leaves the cut to a call of its own, so that the host may say what stays in between."""

    def fork(self, src, keep):
        pass

    def cut(self):
        super().fork(0, self.keep)

    def step_then_cut(self, whole):
        """The calls of a step up to the confirmed path's rows, then those of the cut; sequences `whole` keep all their positions."""
        hip = self.hip
        self.parts[0]()
        keep, length = get_i32(hip, self.keep, self.NSEQ), get_i32(hip, self.len, self.NSEQ)
        hip.htod(np.where(whole, length, keep).astype(np.int32), self.keep)
        self.parts[1]()


@pytest.mark.parametrize("graph", [False, True])
def test_serving_chunks_beside_trees(hip, graph):
    """Chunks of a prompt of no more rows than a tree has, as trees without branches beside drafted ones: all of their positions stay, the
    choice after the last chunk is the one after its last row, and the sequence goes on with trees. Eager and as two recorded parts."""
    rng = np.random.default_rng(21)
    sv = PartsServer(hip, 10)
    prompts = [rng.integers(0, sv.vocab, k) for k in (5, 17, 15, 4)]
    truth = plain_tokens(hip, 10, prompts, 50)
    n, first = sv.NSEQ, [5, 17, 1, 4]  # (14 of the third prompt's tokens come in chunks)
    sv.inputs(np.concatenate([p[:k] for p, k in zip(prompts, first)]))
    hip.htod(np.array(first, np.int32), sv.add)
    sv.layer(sum(first), max(first))
    toks, got = [p[:k].tolist() for p, k in zip(prompts, first)], [[truth[s][0]] if first[s] == len(prompts[s]) else [] for s in range(n)]
    sv.parts = (sv.step, sv.cut)
    graphs, cut_short = [], 0
    for k in range(7):
        chunk = min(NODES - (k == 0), len(prompts[2]) - len(toks[2])) if not got[2] else 0
        sizes = [chunk if s == 2 and chunk else int(rng.integers(2, NODES + 1)) for s in range(n)]
        trees = [draft(rng, truth[s], len(got[s]), q, sv.vocab) if got[s] else (list(range(-1, q - 1)), prompts[s][len(toks[s]):len(toks[s]) + q].tolist()) for s, q in enumerate(sizes)]
        parent, tokens = (np.concatenate([np.array(tr[i], np.int64) for tr in trees] + [np.zeros(sv.t, np.int64)])[:sv.t] for i in (0, 1))
        sv.inputs(tokens)
        for v, b in ((sizes, sv.add), (parent, sv.parent), (tokens, sv.tokens)):
            hip.htod(np.asarray(v, np.int32), b)
        if graph and k == 1:  # (the step before has sized the workspace)
            graphs = [hip.record_graph(f, keep=[sv]) for f in sv.parts]
            sv.parts = [g.launch for g in graphs]
        sv.step_then_cut(np.array([s == 2 and chunk > 0 for s in range(n)]))
        n_path, chosen = get_i32(hip, sv.n_path, n), get_i32(hip, sv.chosen, n * PATH).reshape(n, PATH)
        ids, q_start = get_i32(hip, sv.row_ids, sv.t), np.concatenate([[0], np.cumsum(sizes)])
        for s in range(n):
            if s == 2 and chunk:
                cut_short += n_path[s] < chunk
                toks[s] = toks[s] + prompts[s][len(toks[s]):len(toks[s]) + chunk].tolist()
                if len(toks[s]) == len(prompts[s]):
                    assert ids[q_start[s + 1] - 1] == truth[s][0]
                    got[s] = [truth[s][0]]
                continue
            c = int(n_path[s])
            assert chosen[s, :c].tolist() == truth[s][len(got[s]):len(got[s]) + c], (k, s)
            toks[s] = toks[s] + [got[s][-1]] + chosen[s, :c - 1].tolist()
            got[s] = got[s] + chosen[s, :c].tolist()
        sv.check_pool()
        sv.check_cache(toks)
    assert cut_short and len(got[2]) > 2 and get_i32(hip, sv.err, 1)[0] == 0
    for g in graphs:
        g.close()
