"""The operators for drafted trees and branching sequences, through the C ABI, against their plain restatements
(tests/branch_oracle.py): positions, masks, paths, page tables and moved rows bit for bit, attention and log probabilities against
float64."""
import numpy as np
import pytest

import rustingstrata_amd as S
from tests import branch_oracle as B
from tests import serve_oracle as V
from tests.helpers import rel_l2
from tests.test_gpu_serve import GUARD, Batch, get_i32, i32, up

pytestmark = pytest.mark.gpu


def random_tree(rng, n, shape="any"):
    """Parents of n rows: row 0 the root, a parent before its children."""
    if shape == "line":
        return [i - 1 for i in range(n)]
    if shape == "star":
        return [-1] + [0] * (n - 1)
    return [-1] + [int(i * rng.random() ** (3 if shape == "bushy" else 1)) for i in range(1, n)]


def guarded(hip, n):
    return i32(hip, [GUARD] * (n + 1))


def check_i32(hip, buf, want, name=""):
    want = np.asarray(want).reshape(-1)
    got = get_i32(hip, buf, want.size + 1)
    np.testing.assert_array_equal(got[:-1], want.astype(np.int64).astype(np.uint32).astype(np.int32) if name == "mask" else want, err_msg=name)
    assert got[-1] == GUARD, name


# ---------------- positions and masks ----------------
@pytest.mark.parametrize("words", [1, 2, 3, 4, 5, 8])
@pytest.mark.parametrize("shape", ["any", "line", "star", "bushy"])
def test_tree_step(hip, words, shape):
    """Trees of one node to the most, sequences without rows, lines of more rows than bits, rows behind the last sequence."""
    rng = np.random.default_rng(words)
    sizes = [1, 0, 32 * words, 32 * words + 1, 2, 31, 0, 32 * words - 1, 200, 1] + rng.integers(1, 32 * words + 1, 30).tolist()
    q_start = np.concatenate([[0], np.cumsum(sizes)])
    t, t_max = q_start[-1], q_start[-1] + 70
    parent = np.concatenate([random_tree(rng, n, shape) for n in sizes if n] + [np.full(70, 9)])
    length = np.array(sizes) + rng.integers(0, 3000, len(sizes)) * (rng.random(len(sizes)) < 0.8)
    P = 0 if words == 2 else 1234
    pos, mask = guarded(hip, t_max), guarded(hip, t_max * words)
    hip.tree_step(len(sizes), i32(hip, q_start), i32(hip, parent), i32(hip, length), t_max, words, pos, mask, prefix_len=i32(hip, [P]) if P else 0)
    want, bits, bad = B.tree_step(q_start, parent, length, P, t_max, words)
    assert bad == 0 and (want[t:] == -1).all()
    check_i32(hip, pos, want, "pos")
    check_i32(hip, mask, bits, "mask")


def test_tree_step_of_bad_parents(hip):
    """Parents that are not below their rows are roots and are counted; rows past t, lengths below the rows, positions past 31 bits."""
    rng = np.random.default_rng(3)
    q_start, t = [0, 40, 70, 71, 300], 110
    parent = rng.integers(-40, 60, t)
    parent[5], parent[6] = 2**31 - 1, -2**31
    length, err = [10, 2**31 - 1, -7, 3], i32(hip, [5])
    pos, mask = guarded(hip, t), guarded(hip, 2 * t)
    hip.tree_step(4, i32(hip, q_start), i32(hip, parent), i32(hip, length), t, 2, pos, mask, prefix_len=i32(hip, [100]), err=err)
    want, bits, bad = B.tree_step(q_start, parent, length, 100, t, 2)
    assert bad > 20 and want[40:70].max() == 2**31 - 1
    check_i32(hip, pos, want, "pos")
    check_i32(hip, mask, bits, "mask")
    assert get_i32(hip, err, 1)[0] == 5 + bad


def test_tree_step_of_row_starts_past_the_rows(hip):
    """Row starts that say more than there is, up to 2^31 - 1: nothing is written past the t rows or before them."""
    t = 40
    parent = [-1 if i < 1 else i - 1 for i in range(t)]
    for q_start in ([0, 5, 2**31 - 1], [2**31 - 1] * 3, [-5, 9, 2**31 - 200], [-2**31, -1, 17]):
        pos, mask = i32(hip, [GUARD] * (2 * t + 1)), i32(hip, [GUARD] * (2 * t + 1))
        hip.tree_step(2, i32(hip, q_start), i32(hip, parent), i32(hip, [70, 60]), t, 1, int(pos) + 4 * t, int(mask) + 4 * t)
        want, bits, _ = B.tree_step(q_start, parent, [70, 60], 0, t, 1)
        written = np.zeros(t, bool)  # (rows of no sequence, before the end that the starts give, are left as they are)
        written[min(max(q_start[2], 0), t):] = True
        for s in range(2):
            written[min(max(q_start[s], 0), t):min(max(q_start[s + 1], 0), t)] = True
        for b, w in ((pos, want), (mask, bits[:, 0].astype(np.int64).astype(np.uint32).astype(np.int32))):
            got = get_i32(hip, b, 2 * t + 1)
            assert (got[:t] == GUARD).all() and got[-1] == GUARD
            np.testing.assert_array_equal(got[t:-1], np.where(written, w, GUARD))


# ---------------- the confirmed path ----------------
def accept_case(rng, sizes, words, agree, vocab=50):
    q_start = np.concatenate([[0], np.cumsum(sizes)])
    t = int(q_start[-1])
    parent = np.concatenate([random_tree(rng, n, rng.choice(["any", "line", "star", "bushy"])) for n in sizes if n] + [[]]).astype(np.int64)
    tokens, ids = rng.integers(0, vocab, t), rng.integers(0, vocab, t)
    for s in range(len(sizes)):
        for r in range(q_start[s] + 1, q_start[s + 1]):
            if rng.random() < agree:
                ids[q_start[s] + parent[r]] = tokens[r]
    slots = rng.permutation(5 * t + 5)[:t]
    length = np.array(sizes) + rng.integers(0, 500, len(sizes))
    return q_start, parent, tokens, ids, length, slots


@pytest.mark.parametrize("words,max_path", [(1, 1), (1, 5), (1, 32), (2, 64), (2, 7), (3, 96), (4, 128), (8, 256)])
@pytest.mark.parametrize("agree", [0.0, 0.5, 1.0])
def test_tree_accept(hip, words, max_path, agree):
    """Paths of one row to the whole tree, equal tokens among siblings, choices of none, refused sequences, lines, no rows."""
    rng = np.random.default_rng(words + max_path)
    sizes = [1, 0, 32 * words, 32 * words + 1, 2, 32 * words, 300, 0, 32 * words - 1] + rng.integers(1, 32 * words + 1, 40).tolist()
    q_start, parent, tokens, ids, length, slots = accept_case(rng, sizes, words, agree, vocab=5 if max_path == 7 else 50)
    ids[rng.random(len(ids)) < 0.03] = -1
    slots[q_start[4]], slots[rng.random(len(slots)) < 0.02] = -1, -1
    n, dev = len(sizes), [i32(hip, v) for v in (q_start, parent, tokens, ids, length, slots)]
    out = [guarded(hip, k) for k in (n, n * max_path, n, n, 3 * n * max_path)]
    hip.tree_accept(n, *dev, len(ids), words, max_path, *out)
    want = B.tree_accept(q_start, parent, tokens, ids, length, slots, words, max_path)
    assert agree < 1 or max(want["n_path"]) >= min(max_path, 10)
    for b, name in zip(out, ("n_path", "chosen", "last", "keep", "runs")):
        check_i32(hip, b, want[name], name)


# ---------------- forks ----------------
class Fork:
    def __init__(self, hip, length, tables, page, max_pages, free, n_free, n_pages, refs, src=None, keep=None, place=False):
        B_ = len(length)
        self.hip, self.nseq, self.page, self.max_pages, self.n_pages = hip, B_, page, max_pages, n_pages
        self.src, self.keep = (i32(hip, v) if v is not None else 0 for v in (src, keep))
        self.len, self.n_free = i32(hip, np.append(length, GUARD)), i32(hip, [n_free, GUARD])
        self.tables, self.free, self.refs = (i32(hip, np.append(v, GUARD)) for v in (tables, free, refs))
        self.len_out, self.n_free_out = (self.len, self.n_free) if place else (guarded(hip, B_), guarded(hip, 1))
        self.runs, self.err = guarded(hip, 3 * B_), i32(hip, [5])

    def run(self):
        self.hip.kv_pages_fork(self.nseq, self.src, self.keep, self.len, self.tables, self.max_pages, self.page, self.free, self.n_pages, self.n_free,
                               self.refs, self.len_out, self.n_free_out, self.runs, err=self.err)
        return self

    def check(self, want):
        for name in ("tables", "free", "refs", "len_out", "n_free_out", "runs"):
            check_i32(self.hip, getattr(self, name), want[name], name)
        assert get_i32(self.hip, self.err, 1)[0] == 5 + want["refused"]


def pool_case(rng, nseq, page, max_pages, spare):
    """Sequences that share the pages of a few stems, and own the rest."""
    limit = max_pages * page
    length = np.where(rng.random(nseq) < 0.1, 0, rng.integers(0, limit + 1, nseq))
    stems = [(rng.integers(0, max_pages + 1)) for _ in range(max(1, nseq // 4))]
    n_pages = sum(stems) + nseq * max_pages + spare
    order, at = rng.permutation(n_pages), 0
    rows = []
    for k in stems:
        rows.append(order[at:at + k])
        at += k
    tables, refs = rng.integers(-3, n_pages + 3, (nseq, max_pages)), np.full(n_pages, 0)
    count = np.zeros(n_pages, np.int64)
    for s in range(nseq):
        stem, have = rows[rng.integers(0, len(rows))], -(-length[s] // page)
        k = min(len(stem), length[s] // page)  # (only full pages are shared)
        tables[s, :k] = stem[:k]
        tables[s, k:have] = order[at:at + have - k]
        at += have - k
        count[tables[s, :have]] += 1
    free = np.concatenate([order[at:], rng.integers(0, n_pages, at)])  # (behind the unused pages: anything)
    refs = np.maximum(count - 1, 0)
    # the stems' pages that nobody holds are free as well
    unused = [p for stem in rows for p in stem if not count[p]]
    n_free = n_pages - at
    free[n_free:n_free + len(unused)] = unused
    return length, tables, free, n_free + len(unused), n_pages, refs


@pytest.mark.parametrize("nseq,page,max_pages,spare", [(1, 16, 3, 2), (5, 64, 1, 3), (16, 16, 7, 40), (17, 16, 7, 40), (64, 32, 70, 9), (257, 16, 5, 3), (1030, 16, 4, 600), (4096, 16, 3, 2000)])
@pytest.mark.parametrize("what", ["both", "beams", "cut", "end", "none", "swap"])
def test_pages_fork(hip, nseq, page, max_pages, spare, what):
    """Every output, the tables, the stack and the holders' counts, in one launch and in four, with sequences refused for want of
    pages; in place as well as not."""
    rng = np.random.default_rng(nseq + len(what))
    length, tables, free, n_free, n_pages, refs = pool_case(rng, nseq, page, max_pages, spare)
    if what in ("both", "end"):
        n_free = min(n_free, nseq // 5)
    src = dict(both=rng.integers(0, nseq, nseq), beams=rng.integers(0, nseq, nseq) // 4 * 4, swap=rng.permutation(nseq)).get(what)
    keep = dict(both=rng.integers(0, max_pages * page + 1, nseq), cut=length - rng.integers(0, 40, nseq), end=np.where(rng.random(nseq) < 0.3, 0, length)).get(what)
    want = B.pages_fork(src, keep, length, tables, max_pages, page, free, n_pages, n_free, refs)
    assert nseq < 64 or (want["refused"] > 0) == (what == "both") or what in ("cut", "beams")
    for place in (False, True):
        Fork(hip, length, tables, page, max_pages, free, n_free, n_pages, refs, src, keep, place).run().check(want)


def full_pool(rng, length, page, max_pages):
    """Sequences of these lengths, each next to the one before sharing a random part of its full pages, over a pool of just their pages."""
    nseq, rows, at = len(length), np.full((len(length), max_pages), -1), 0
    for s, n in enumerate(length):
        have = -(-n // page)
        k = min(int(rng.integers(0, max_pages)), n // page, length[s - 1] // page) if s and rng.random() < 0.3 else 0
        rows[s, :k] = rows[s - 1, :k]
        rows[s, k:have] = np.arange(at, at + have - k)
        at += have - k
    order = rng.permutation(at)
    tables = np.where(rows >= 0, order[np.maximum(rows, 0)], rng.integers(-3, at + 3, rows.shape))
    return length, tables, rng.integers(0, at, at), 0, at, np.maximum(np.bincount(order[rows[rows >= 0]], minlength=at) - 1, 0)


@pytest.mark.parametrize("nseq", [9, 300])
def test_pages_fork_of_anything(hip, nseq):
    """Lengths, sources, page ids, counts and stacks outside their limits."""
    rng = np.random.default_rng(nseq)
    length, tables, free, n_free, n_pages, refs = pool_case(rng, nseq, 16, 4, 5)
    length[rng.random(nseq) < 0.2] = -5
    length[rng.random(nseq) < 0.1] = 2**31 - 1
    tables[rng.random(tables.shape) < 0.1] = -1
    tables[rng.random(tables.shape) < 0.1] = n_pages
    free[rng.random(n_pages) < 0.3] = 2**31 - 1
    src, keep = rng.integers(-2, nseq + 2, nseq), rng.integers(-9, 80, nseq)
    keep[0], keep[1], src[2] = 2**31 - 1, -2**31, 2**31 - 1
    for n in (n_free, -3, 2**31 - 1):
        want = B.pages_fork(src, keep, length, tables, 4, 16, free, n_pages, n, refs)
        assert want["refused"] > 0
        Fork(hip, length, tables, 16, 4, free, n, n_pages, refs, src, keep).run().check(want)


@pytest.mark.parametrize("nseq,max_pages", [(256, 128), (32, 1024), (4096, 8), (257, 128), (300, 128), (33, 1024), (4096, 9)])
@pytest.mark.parametrize("what", ["cut", "few", "end", "all", "none"])
def test_pages_fork_of_wide_tables(hip, nseq, max_pages, what):
    """Cuts and ends of a server's sequences without sources, on both sides of the tables that one block takes (2^15 entries): a few
    pages let go and all of them, pages that others hold, cuts refused for want of a page; in place as well as not."""
    page, rng = 16, np.random.default_rng(nseq + len(what))
    length, tables, free, n_free, n_pages, refs = pool_case(rng, nseq, page, max_pages, 40)
    if what == "all":
        length[:] = max_pages * page
        length, tables, free, n_free, n_pages, refs = full_pool(rng, length, page, max_pages)
    keep = dict(cut=rng.integers(0, max_pages * page + 1, nseq), few=length - rng.integers(0, 40, nseq), end=np.where(rng.random(nseq) < 0.3, 0, length), all=np.zeros(nseq, np.int64)).get(what)
    n_free = min(n_free, 5) if what in ("cut", "few") else n_free
    want = B.pages_fork(None, keep, length, tables, max_pages, page, free, n_pages, n_free, refs)
    assert what in ("cut", "few") or want["refused"] == 0
    if what == "all":
        assert want["n_free_out"] == [n_pages] and not want["refs"].any()
    for place in (False, True):
        Fork(hip, length, tables, page, max_pages, free, n_free, n_pages, refs, None, keep, place).run().check(want)


def test_pages_fork_of_nothing(hip):
    Fork(hip, np.zeros(0, int), np.zeros(0, int), 16, 3, np.arange(4), 2, 4, np.zeros(4, int)).run()
    b = i32(hip, [0] * 64)
    for n, want in ((3, 3), (9, 4), (-2, 0)):  # (the stack's height is written all the same)
        out = guarded(hip, 1)
        hip.kv_pages_fork(0, 0, 0, 0, 0, 3, 16, b, 4, i32(hip, [n]), b, 0, out, 0)
        check_i32(hip, out, [want])
    hip.kv_rows_move(b, 0, 16, 4, b, 3, 1)
    hip.kv_rows_move(b, 2, 16, 4, b, 0, 1)


def test_pages_fork_replayed(hip):
    """Forks, cuts and steps of a server's sequences recorded once and replayed: the state follows the restatement."""
    rng = np.random.default_rng(4)
    nseq, page, max_pages, n_pages, t_max = 24, 16, 6, 130, 200
    length, tables, free, n_free, refs = np.zeros(nseq, np.int64), np.zeros((nseq, max_pages), np.int64), rng.permutation(n_pages), n_pages, np.zeros(n_pages, np.int64)
    f = Fork(hip, length, tables, page, max_pages, free, n_free, n_pages, refs, np.arange(nseq), length, place=True)
    add, out = i32(hip, [0] * nseq), [hip.alloc(4 * (k + 1)) for k in (nseq + 1, t_max, t_max)]

    def step():
        f.run()
        hip.kv_pages_step(nseq, add, f.len, f.tables, max_pages, page, f.free, n_pages, f.n_free, t_max, *out, f.len, f.n_free)

    step()
    g = hip.record_graph(step, keep=[f])
    for k in range(40):
        src, keep, more = np.where(rng.random(nseq) < 0.3, rng.integers(0, nseq, nseq), np.arange(nseq)), np.where(rng.random(nseq) < 0.4, rng.integers(0, 80, nseq), 10**6), rng.integers(0, 9, nseq)
        want = B.pages_fork(src, keep, length, tables, max_pages, page, free, n_pages, n_free, refs)
        d = V.pages_step(more, want["len_out"], want["tables"], max_pages, page, want["free"], n_pages, want["n_free_out"][0], 0, t_max)
        for v, b in ((src, f.src), (keep, f.keep), (more, add), ([5], f.err)):
            hip.htod(np.asarray(v, np.int32), b)
        g.launch()
        f.check(dict(want, tables=d["tables"], free=d["free"], len_out=d["len_out"], n_free_out=[d["n_free_out"]]))
        length, tables, free, n_free, refs = np.array(d["len_out"]), d["tables"], d["free"], d["n_free_out"], want["refs"]
    g.close()


# ---------------- rows of the caches ----------------
@pytest.mark.parametrize("row_bytes", [16, 128, 272, 1024, 4096, 5008])
@pytest.mark.parametrize("caches", [1, 5])
def test_rows_move(hip, row_bytes, caches):
    """Rows that close up over rows already read, runs of many rows, runs that leave the caches, empty groups."""
    rng = np.random.default_rng(row_bytes)
    n_slots, per, groups = 1200, 70, 9
    data = rng.integers(-2**31, 2**31, (caches, n_slots, row_bytes // 4)).astype(np.int32)
    runs = np.zeros((groups, per, 3), np.int64)
    for g in range(groups):
        base = 110 * g
        kind = g % 3
        if kind == 0:  # a path closing up: row path[i] to place i
            path = np.concatenate([[0], np.sort(rng.choice(np.arange(1, 100), per - 1, replace=False))])
            runs[g] = np.stack([base + path, base + np.arange(per), path != np.arange(per)], 1)
        elif kind == 1:  # runs of many rows, one past another
            runs[g, 3], runs[g, 5], runs[g, 69] = (base, base + 60, 37), (base + 38, base + 97, 3), (base + 41, base + 100, 9)
        runs[g, 30 if kind else 0] = [(-1, base, 2), (base, n_slots - 1, 2), (base, base + 5, -3), (n_slots, base, 1), (base, -2**31, 2**31 - 1)][g % 5]
    if groups > 2:
        runs[2] = 0
    want = np.stack([B.rows_move(c.copy(), runs, n_slots) for c in data])
    bufs = [up(hip, np.concatenate([c.reshape(-1), [GUARD]]).astype(np.int32)) for c in data]
    table = up(hip, np.array([int(b) for b in bufs], np.uint64))
    hip.kv_rows_move(table, caches, row_bytes, n_slots, i32(hip, runs), groups, per)
    for b, w in zip(bufs, want):
        check_i32(hip, b, w)


def test_rows_move_of_more_blocks_than_one_launch(hip):
    """2^20 groups of 17 caches, more than 2^24 pieces of work: runs of the first and the last groups and of those on both sides of
    every 2^23rd piece, eager and recorded."""
    groups, caches, n_slots, row_bytes = 1 << 20, 17, 64, 16
    rng = np.random.default_rng(1)
    data = rng.integers(-2**31, 2**31, (caches, n_slots, row_bytes // 4)).astype(np.int32)
    runs = np.zeros((groups, 1, 3), np.int32)
    busy = sorted({0, 1, groups - 2, groups - 1} | {(k << 23) // caches + d for k in (1, 2) for d in (-1, 0, 1)})
    for i, g in enumerate(busy):  # (no run reads a row that another writes)
        runs[g, 0] = i, 32 + 2 * i, 1 + i % 2
    bufs = [up(hip, np.concatenate([c.reshape(-1), [GUARD]]).astype(np.int32)) for c in data]
    table, moves = up(hip, np.array([int(b) for b in bufs], np.uint64)), up(hip, runs)
    call = lambda: hip.kv_rows_move(table, caches, row_bytes, n_slots, moves, groups, 1)  # noqa: E731
    g = hip.record_graph(call, keep=[table, moves, *bufs])
    for run in (call, g.launch):
        for b, c in zip(bufs, data):
            hip.htod(c, b)
        run()
        for b, c in zip(bufs, data):
            check_i32(hip, b, B.rows_move(c.copy(), runs[busy].astype(np.int64), n_slots))
    g.close()


@pytest.mark.parametrize("groups,caches,per", [(300, 13, 7), (2100, 1, 2), (700, 3, 64), (260, 9, 65), (150, 16, 256), (90, 30, 129)])
def test_rows_move_of_many_caches(hip, groups, caches, per):
    """Groups and caches enough for a block to take several caches, the last one fewer, and runs of 2 to 256 a group: paths that close
    up, each in slots of its own."""
    rng = np.random.default_rng(per)
    row_bytes, room = 32, per + 3
    n_slots = groups * room
    data = rng.integers(-2**31, 2**31, (caches, n_slots, row_bytes // 4)).astype(np.int32)
    runs = np.zeros((groups, per, 3), np.int64)
    for g in range(groups):
        k = int(rng.integers(0, per + 1))
        path = np.sort(rng.choice(room, k, replace=False))
        runs[g, :k] = np.stack([g * room + path, g * room + np.arange(k), path != np.arange(k)], 1)
    want = np.stack([B.rows_move(c.copy(), runs, n_slots) for c in data])
    bufs = [up(hip, np.concatenate([c.reshape(-1), [GUARD]]).astype(np.int32)) for c in data]
    hip.kv_rows_move(up(hip, np.array([int(b) for b in bufs], np.uint64)), caches, row_bytes, n_slots, i32(hip, runs), groups, per)
    for b, w in zip(bufs, want):
        check_i32(hip, b, w)


def test_rows_move_of_a_whole_page(hip):
    """One run a group, longer than a batch, to another page."""
    rng = np.random.default_rng(1)
    for row_bytes, n in ((1024, 1000), (128, 3000), (64, 257)):
        data = rng.integers(-2**31, 2**31, (2 * n + 3, row_bytes // 4)).astype(np.int32)
        runs = np.array([[[1, n + 2, n]]])
        b = up(hip, data)
        hip.kv_rows_move(up(hip, np.array([int(b)], np.uint64)), 1, row_bytes, len(data), i32(hip, runs), 1, 1)
        np.testing.assert_array_equal(hip.get(b, np.int32, data.size).reshape(data.shape), B.rows_move(data.copy(), runs, len(data)))


def test_rows_move_offsets_past_32_bits(hip):
    """A cache of more than 4 GiB."""
    row, n_slots = 1 << 20, 4200
    b = hip.alloc(row * n_slots)
    marks = np.random.default_rng(2).integers(-2**31, 2**31, (3, row // 4)).astype(np.int32)
    for i, m in enumerate(marks):
        hip.htod(m, int(b) + (4190 + i) * row)
    hip.kv_rows_move(up(hip, np.array([int(b)], np.uint64)), 1, row, n_slots, i32(hip, [4190, 3, 2, 4192, 4195, 1]), 1, 2)
    for at, m in ((3, marks[0]), (4, marks[1]), (4195, marks[2]), (4191, marks[1])):
        np.testing.assert_array_equal(hip.get(int(b) + at * row, np.int32, row // 4), m)


# ---------------- log probabilities ----------------
def logits(rows, n, seed, kind="normal"):
    rng = np.random.default_rng(seed)
    x = (4 * rng.standard_normal((rows, n))).astype(np.float32)
    if kind == "masked":
        x[rng.random((rows, n)) < np.where(np.arange(rows) % 3 == 0, 1.0, np.where(np.arange(rows) % 3 == 1, 0.999, 0.5))[:, None]] = -np.inf
    elif kind == "ties":
        x = np.round(x).astype(np.float32)
        x[rng.random((rows, n)) < 0.2] = -0.0
    elif kind == "sorted":
        x = np.sort(x, 1)
        x[::2] = x[::2, ::-1]
    elif kind == "wide":
        x *= np.float32(10) ** rng.integers(-30, 38, (rows, 1)).astype(np.float32)
        x[:, ::7] = np.finfo(np.float32).min
    elif kind == "special":
        x[0, 0], x[rows // 2, n // 2], x[rows - 1, n - 1] = np.nan, np.inf, -np.inf
        x[rows // 3, n // 3] = np.array([0xFFC00001], np.uint32).view(np.float32)[0]
    elif kind == "same":
        x[:] = np.float32(-2.5)
    return x


class Logp:
    def __init__(self, hip, x, ids, k, stride=None, shift=0, rank=True):
        rows, n = x.shape
        stride = stride or n
        buf = np.full(shift + rows * stride + 3, np.float32(np.nan))
        for r in range(rows):
            buf[shift + r * stride:shift + r * stride + n] = x[r]
        self.hip, self.x, self.ids_, self.k, self.m = hip, x, ids, k, ids.shape[1]
        self.b, self.at, self.stride = up(hip, buf), 4 * shift, stride
        self.ids = i32(hip, ids) if self.m else 0
        self.logp, self.entropy, self.top_logp = (up(hip, np.full(v + 1, 6.5, np.float32)) for v in (rows * self.m, rows, rows * k))
        self.rank, self.top_ids, self.with_rank = guarded(hip, rows * self.m), guarded(hip, rows * k), rank

    def run(self):
        rows, n = self.x.shape
        self.hip.logits_logprobs(int(self.b) + self.at, self.stride, n, rows, ids=self.ids, m=self.m, logp=self.logp, rank=self.rank if self.with_rank else 0,
                                 entropy=self.entropy, k=self.k, top_ids=self.top_ids, top_logp=self.top_logp)
        return self

    def get(self):
        rows, hip = len(self.x), self.hip
        return (*(hip.get(b, np.float32, v + 1) for b, v in ((self.logp, rows * self.m), (self.entropy, rows), (self.top_logp, rows * self.k))), get_i32(hip, self.rank, rows * self.m + 1),
                get_i32(hip, self.top_ids, rows * self.k + 1))

    def check(self):
        """In units of 2^-24: a term e^y of S has an exponent that is off by 3 |y| (the difference, log2 e and the product), and the
        mean of |y| over S's terms is at most ln n; its exp adds 2, a thread's additions one a tile (n / 4096) and 4, and 14 joins 4
        each: S is within `sums` of itself. ln S adds S's error and its own rounding, the difference x - M and the last subtraction
        one rounding each. The entropy's W / S has terms up to ln n times as large."""
        n = self.x.shape[1]
        logp, rank, entropy, top_ids, top_logp = B.logprobs(self.x, self.ids_, self.k)
        got_logp, got_h, got_top, got_rank, got_ids = self.get()
        assert got_logp[-1] == got_h[-1] == got_top[-1] == np.float32(6.5)
        sums = 2.0 ** -24 * (3 * np.log(n) + n / 4096 + 62)
        for got, want in ((got_logp[:-1], logp), (got_top[:-1], top_logp)):
            want = want.reshape(-1)
            np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
            fine = np.isfinite(want) & (np.abs(want) < 3.1e38)  # (a difference past float32's range is -inf)
            assert (got[~fine & ~np.isnan(want)] <= -3e38).all()
            assert (np.abs(got[fine] - want[fine]) <= 2.0 ** -22 * (np.abs(want[fine]) + np.log(n)) + sums).all()
        np.testing.assert_array_equal(np.isnan(got_h[:-1]), np.isnan(entropy))
        fine = np.isfinite(entropy)
        assert (np.abs(got_h[:-1][fine] - entropy[fine]) <= 2.0 ** -22 * np.log(n + 1) + (1 + np.log(n)) * sums).all()
        if self.with_rank:
            np.testing.assert_array_equal(got_rank, np.append(rank.reshape(-1), GUARD))
        np.testing.assert_array_equal(got_ids, np.append(top_ids.reshape(-1), GUARD))


@pytest.mark.parametrize("rows,n,m,k", [(1, 1, 1, 1), (1, 3, 2, 5), (2, 255, 0, 3), (3, 4095, 1, 64), (3, 4096, 1, 0), (1, 4097, 3, 20), (5, 20001, 16, 1), (2, 151936, 1, 20), (40, 32003, 4, 5), (130, 9001, 5, 64),
                                        (1030, 1001, 1, 7), (1500, 37, 1, 64)])
@pytest.mark.parametrize("kind", ["normal", "masked", "ties", "sorted", "wide", "special", "same"])
def test_logprobs(hip, rows, n, m, k, kind):
    """One row to many, rows in parts and whole, rows that begin at any 4 bytes; masked, tied, sorted and special logits; ids outside."""
    rng = np.random.default_rng(n)
    x = logits(rows, n, rows + n, kind)
    ids = rng.integers(0, n, (rows, m))
    if m > 1:
        ids[:, 1] = np.argmax(np.where(np.isnan(x), -np.inf, x), 1)
        ids[0, 0], ids[rows - 1, 1] = -1, n
    Logp(hip, x, ids, k).run().check()
    if kind in ("normal", "ties", "masked"):
        Logp(hip, x, ids, k, stride=n + 1, shift=3, rank=False).run().check()
        Logp(hip, x, ids, k, stride=n + 5, shift=1).run().check()


@pytest.mark.parametrize("rows,n", [(1, 5), (2, 9001), (600, 9001), (1, 50001)])
def test_logprobs_ranks_at_the_ends_of_the_order(hip, rows, n):
    """Given tokens that are the greatest and the least of all values (the NaN whose bits are 0x7FFFFFFF, and 0xFFFFFFFF), alone and
    twice, at the first, a middle and the last index, beside tokens around them."""
    rng = np.random.default_rng(n)
    x = logits(rows, n, n)
    for r in range(rows):
        at = [0, n // 2, n - 1]
        top, low = int(rng.integers(0, 3)), int(rng.integers(0, 3))
        bits = x[r].view(np.uint32)
        bits[at[top]] = 0x7FFFFFFF
        if r % 3 == 1:
            bits[at[(top + 1) % 3]] = 0x7FFFFFFF
        if low != top:
            bits[at[low]] = 0xFFFFFFFF
        if r % 3 == 2:
            bits[min(n - 1, n // 2 + 3)] = 0xFFFFFFFF
    ids = np.stack([np.full(rows, v) for v in (0, n // 2, n - 1, 1, min(n - 1, n // 2 + 3), max(0, n - 2), -1, n)], 1)
    Logp(hip, x, ids, 4).run().check()
    Logp(hip, x, ids, 0, stride=n + 2, shift=1).run().check()
    for i in range(ids.shape[1]):
        Logp(hip, x, ids[:, i:i + 1], 0).run().check()


def test_logprobs_of_rising_rows(hip):
    """Whole rows of many tiles in rising order, so that the waves agree on another bound each time; every call gives the same bits."""
    x = np.sort(logits(520, 70001, 3), 1)
    x[1::3, ::9] = x[1::3, 40000:40001]
    c = Logp(hip, x, np.full((520, 1), 70000), 64).run()
    c.check()
    want = c.get()
    for _ in range(5):
        for a, b in zip(c.run().get(), want):
            np.testing.assert_array_equal(a, b)


def test_logprobs_parts_alone(hip):
    """Each output alone gives what all together do."""
    x, ids = logits(7, 30001, 5), np.random.default_rng(1).integers(0, 30001, (7, 2))
    both = Logp(hip, x, ids, 9).run().get()
    for i, name in enumerate(("logp", "entropy", "top_logp", "rank", "top_ids")):
        c = Logp(hip, x, ids, 9)
        hip.logits_logprobs(c.b, 30001, 30001, 7, ids=c.ids, m=2, k=9, **{name: getattr(c, name)})
        np.testing.assert_array_equal(c.get()[i], both[i])


def test_logprobs_replayed(hip):
    """Two graphs of one context (few rows in parts, many whole) beside eager calls: every replay gives the eager bits."""
    rng = np.random.default_rng(6)
    cases = [Logp(hip, logits(r, n, r), rng.integers(0, n, (r, 1)), k) for r, n, k in ((3, 50001, 20), (1200, 300, 5))]
    want = []
    for c in cases:
        c.run()
        want.append(c.get())
    graphs = [hip.record_graph(c.run, keep=[c]) for c in cases]
    for k in range(4):
        for c in cases:
            for b, v in ((c.logp, 6.5), (c.entropy, 6.5), (c.top_logp, 6.5)):
                hip.htod(np.full(1, v, np.float32), b)
        for g in graphs[::1 if k % 2 else -1]:
            g.launch()
        for c, w in zip(cases, want):
            for a, b in zip(c.get(), w):
                np.testing.assert_array_equal(a, b)
        cases[k % 2].run()
    for g in graphs:
        g.close()


def test_logprobs_of_the_longest_row(hip):
    """A row of 2^31 - 1 logits: the last one is the likeliest."""
    n = 2**31 - 1
    x = hip.alloc(4 * n)
    hip.memset(x, 4 * n)
    hip.htod(np.array([30.0], np.float32), int(x) + 4 * (n - 1))
    hip.htod(np.array([25.0], np.float32), int(x) + 4 * 12345)
    ids, rank, logp, top = i32(hip, [n - 1, 0]), guarded(hip, 2), up(hip, np.zeros(2, np.float32)), guarded(hip, 3)
    h = up(hip, np.zeros(1, np.float32))
    hip.logits_logprobs(x, n, n, 1, ids=ids, m=2, logp=logp, rank=rank, entropy=h, k=3, top_ids=top)
    check_i32(hip, top, [n - 1, 12345, 0])
    check_i32(hip, rank, [1, 3])
    s = 1 + np.exp(-5.0) + (n - 2) * np.exp(-30.0)
    want = np.array([-np.log(s), -30 - np.log(s)])
    assert np.abs(hip.get(logp, np.float32, 2) - want).max() <= 2.0 ** -19


# ---------------- attention ----------------
class Trees(Batch):
    """Batch whose sequences' rows are trees; room: pages that a table has room for at least (many: the call's bounds allow much
    work, which takes another form)."""

    def __init__(self, hip, q, n, nh, nkv, hd, page, words, P=0, seed=0, shape="any", room=0, **kw):
        super().__init__(hip, q, n, nh, nkv, hd, page, P=P, seed=seed, **kw)
        rng = np.random.default_rng(seed + 1000)
        if room > self.max_pages:
            self.tables = np.concatenate([self.tables, rng.integers(-5, self.n_pages + 5, (self.nseq, room - self.max_pages))], 1)
            self.max_pages = room
        self.words = words
        self.parent = np.concatenate([random_tree(rng, k, shape) for k in q if k] + [np.full(kw.get("extra", 0), -1)]).astype(np.int64)
        self.pos, self.mask, _ = B.tree_step(self.q_start, self.parent, self.n, P, self.t, words)

    def upload(self):
        super().upload()
        self.b["mask"] = up(self.hip, self.mask)
        return self

    def launch(self, win=0, max_prefix=None, max_q=None):
        mp = self.P if max_prefix is None else max_prefix
        p = dict(self.pb) if mp else dict(sink=self.pb["sink"])
        self.hip.attn_paged_tree(out=self.out, t=self.t, max_q=max_q or self.max_q, nseq=self.nseq, max_pages=self.max_pages, page=self.page,
                                 n_pages=self.n_pages, nh=self.nh, nkv=self.nkv, hd=self.hd, scale=self.scale, max_prefix=mp, win=win, words=self.words, **self.b, **p)

    def want(self, win=0, rows=None):
        return B.attn_tree(self.q, self.kc, self.vc, self.pos, self.mask, self.q_start, self.n, self.tables, self.page, self.prefix, self.P, self.scale, self.words,
                           win=win, sink=self.sink, gate=self.gate[:, :, 1] if self.gate is not None else None, rows=rows)


SHAPES = [(8, 1, 128), (8, 2, 64), (4, 2, 128), (4, 4, 64), (3, 3, 128)]


@pytest.mark.parametrize("nh,nkv,hd", SHAPES)
@pytest.mark.parametrize("P,win", [(0, 0), (0, 40), (70, 0), (333, 100)])
@pytest.mark.parametrize("most,room", [(2, 0), (4, 0), (9, 0), (32, 0), (9, 6000), (32, 6000)])
def test_attn_tree(hip, nh, nkv, hd, P, win, most, room):
    """Trees of 1 to `most` nodes over 0 to 700 keys around the borders of pages and tiles, sequences without rows, rows behind the
    last sequence."""
    rng = np.random.default_rng(most + P)
    before = [0, 0, 1, 15, 16, 31, 33, 63, 64, 65, 127, 129, 300, 700]
    q = [1, most] + rng.integers(1, most + 1, len(before) - 3).tolist() + [0]
    b = Trees(hip, q, [k + m for k, m in zip(before, q)], nh, nkv, hd, 16, 1, P=P, seed=most, sink=P == 70, gate=P == 70, extra=3, big=True, room=room).upload()
    b.launch(win)
    b.check(b.get(), win)


@pytest.mark.parametrize("nh,nkv,hd", SHAPES[:3])
@pytest.mark.parametrize("words,shape", [(2, "any"), (2, "line"), (3, "star"), (5, "bushy"), (8, "any")])
@pytest.mark.parametrize("P", [0, 129])
def test_attn_tree_many_nodes(hip, nh, nkv, hd, words, shape, P):
    """Trees of up to 256 nodes that lie over several tiles of keys, with lines of more rows than bits beside them."""
    most = 32 * words
    q = [most, 1, most - 1, most + 1, 33, 0, most + 60]
    n = [k + b for k, b in zip(q, [0, 5, 64, 100, 31, 77, 200])]
    b = Trees(hip, q, n, nh, nkv, hd, 32, words, P=P, seed=words, shape=shape, gate=words == 3, sink=words == 5, extra=1).upload()
    b.launch()
    b.check(b.get())


def test_attn_tree_long(hip):
    """Trees over long contexts that many blocks share, and over few heads."""
    for nh, nkv, hd, q, before, P in ((8, 1, 128, [26, 3], [20000, 500], 0), (16, 8, 64, [12] * 5, [3000, 1, 2500, 900, 4000], 3000), (32, 4, 128, [64, 64], [9000, 30], 0)):
        b = Trees(hip, q, [k + m for k, m in zip(before, q)], nh, nkv, hd, 64, 2, P=P, seed=nh).upload()
        b.launch()
        b.check(b.get(), rows=sorted(set(range(0, b.t, 7)) | {b.t - 1}))


@pytest.mark.parametrize("nseq", [300, 1030])
@pytest.mark.parametrize("P,hd", [(0, 64), (33, 64), (33, 128)])
def test_attn_tree_many_sequences(hip, nseq, P, hd):
    rng = np.random.default_rng(nseq)
    q = rng.integers(0, 6, nseq).tolist()
    n = [k + int(m) for k, m in zip(q, rng.integers(0, 60, nseq))]
    b = Trees(hip, q, n, 8, 2, hd, 16, 1, P=P, seed=P).upload()
    b.launch()
    b.check(b.get(), rows=sorted(rng.integers(0, b.t, 300).tolist()))


def test_attn_tree_of_lines(hip):
    """Trees without branches: the masks say what the positions do, as attn_paged has it (few rows: its bits)."""
    for q, P in (([1] * 9, 0), ([3, 1, 4], 70), ([20, 1, 17, 2, 32], 0), ([20, 1, 17, 2, 32], 130)):
        b = Trees(hip, q, [k + 40 * i for i, k in enumerate(q)], 8, 2, 128, 16, 1, P=P, seed=P, shape="line").upload()
        b.launch()
        got = b.get()
        b.check(got)
        mask = b.b.pop("mask")
        Batch.launch(b)
        if max(q) <= 8:
            np.testing.assert_array_equal(got, b.get())
        assert rel_l2(got, b.get()) <= 2.0 ** -20
        del mask


@pytest.mark.parametrize("room", [0, 9000])
@pytest.mark.parametrize("q", [[4, 1, 2], [40, 7, 60]])
def test_attn_tree_masks_of_any_bits(hip, q, room):
    """The masks are taken as they are: rows that see nothing of the step, not even themselves; bits of rows behind them do not
    count. Without keys before the rows such a row is 0."""
    for P, before in ((0, 0), (0, 50), (20, 0)):
        b = Trees(hip, q, [k + before for k in q], 8, 2, 64, 16, 2, P=P, seed=7, room=room)
        rng = np.random.default_rng(before)
        b.mask = rng.integers(0, 2**32, b.mask.shape, dtype=np.uint64).astype(np.uint32)
        b.mask[::3] = 0
        b.mask[1::4] = 0xFFFFFFFF
        b.upload().launch()
        got = b.get()
        b.check(got)
        assert P or before or not got[0].any()


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("q,room", [([4, 3], 0), ([30, 40], 0), ([30, 40], 9000)])
def test_attn_tree_non_finite(hip, bad, q, room):
    """Keys and values that are not finite stay out of the rows whose masks do not name them."""
    for P in (0, 70):
        b = Trees(hip, q, [k + 50 for k in q], 8, 2, 64, 16, 2, P=P, seed=3, room=room)
        for s in range(len(q)):  # the last node's key and value: a leaf that no other row sees
            j = b.n[s] - 1
            row = b.tables[s][j // 16] * 16 + j % 16
            b.kc[row], b.vc[row] = bad, bad
        b.upload().launch()
        got = b.get()
        want, top = b.want()
        for r in range(b.t):
            if r + 1 in b.q_start[1:]:
                continue
            for h in range(8):
                assert rel_l2(got[r, h], want[r, h]) <= 2.0 ** -23 * (14 + top[r, h]), (r, h)


@pytest.mark.parametrize("q,room", [([3, 2], 0), ([60, 17], 0), ([60, 17], 9000)])
def test_attn_tree_holes(hip, q, room):
    """Pages outside the pool hold no keys, in the context and under the tree."""
    for P in (0, 90):
        b = Trees(hip, q, [k + 60 for k in q], 8, 1, 128, 16, 2, P=P, seed=5, room=room)
        b.tables[0, 1], b.tables[1, 3], b.tables[0, 3] = -1, b.n_pages, 2**31 - 1
        if P:
            b.prefix[2] = -7
        b.upload().launch()
        b.check(b.get())


def test_attn_tree_offsets_past_32_bits(hip):
    """A pool of 2^22 + slots, more than 2^32 bytes a cache, the sequences on its last pages."""
    b = Trees(hip, [9, 2], [80, 40], 8, 4, 128, 64, 1, seed=2)
    rows, page = 4 * 128, 64
    far = (1 << 32) // (2 * rows) // page + 5
    b2 = dict(kc=hip.alloc((far + b.n_pages) * page * rows * 2), vc=hip.alloc((far + b.n_pages) * page * rows * 2))
    for name, a in (("kc", b.kc), ("vc", b.vc)):
        hip.htod(np.ascontiguousarray(a), int(b2[name]) + far * page * rows * 2)
    b.upload()
    near = b.tables.copy()
    b.b |= dict(kc=b2["kc"], vc=b2["vc"], tables=i32(hip, near + far))
    b.n_pages += far
    b.launch()
    b.n_pages -= far
    b.check(b.get())


@pytest.mark.parametrize("q,room", [([4, 1, 2], 0), ([12, 9, 30], 0), ([40, 70, 3], 0), ([40, 30, 3], 9000)])
def test_attn_tree_prefix_lengths_on_the_device(hip, q, room):
    """A prefix that the call makes room for and the device says is shorter or not there."""
    for P in (1, 50):
        b = Trees(hip, q, [k + 70 for k in q], 8, 2, 64, 16, 2, P=P, seed=8, room=room, sink=True).upload()
        b.launch(max_prefix=4096)
        b.check(b.get())
    b.launch(max_prefix=49)
    less = b.get()
    hip.htod(np.array([49], np.int32), b.pb["prefix_len"])
    b.launch(max_prefix=50)
    np.testing.assert_array_equal(less, b.get())
    a = Trees(hip, q, [k + 70 for k in q], 8, 2, 64, 16, 2, seed=8, room=room, sink=True).upload()
    prefix, none = i32(hip, [0] * 300), i32(hip, [0])
    a.pb |= dict(prefix=prefix, prefix_len=none)
    for n in (0, -5):
        hip.htod(np.array([n], np.int32), none)
        a.launch(max_prefix=4096)
        a.check(a.get())


def test_attn_tree_device_lengths_past_their_bounds(hip):
    """Lengths and row starts that say more than there is, and a sequence whose length does not hold its rows."""
    for q, room in (([4, 3, 2], 0), ([40, 20, 30], 0), ([40, 20, 30], 9000)):
        b = Trees(hip, q, [k + 30 for k in q], 8, 2, 64, 16, 2, seed=4, room=room).upload()
        b.launch()
        want = b.get()
        hip.htod(np.array([2**31 - 1, *b.n[1:]], np.int32), b.b["length"])
        b.launch()
        np.testing.assert_array_equal(b.get()[b.q_start[1]:], want[b.q_start[1]:])
        hip.htod(np.array([1, b.n[1], -5], np.int32), b.b["length"])
        b.launch()
        got = b.get()
        np.testing.assert_array_equal(got[b.q_start[1]:b.q_start[2]], want[b.q_start[1]:b.q_start[2]])
        assert not got[b.q_start[2]:].any()


def test_attn_tree_two_graphs_and_contexts(hip):
    """Graphs of two shapes share the context's workspace; a second context runs the same at once."""
    other = S.HipBackend(0)
    try:
        shapes = (([4] * 6, 0, 0), ([60, 20], 100, 0), ([60, 20], 0, 9000))
        bs = [Trees(h, q, [k + 300 for k in q], 8, 2, 128, 16, 2, P=P, seed=1, room=room).upload() for h in (hip, other) for q, P, room in shapes]
        for b in bs:
            b.launch()
        want = [b.get() for b in bs]
        graphs = [b.hip.record_graph(b.launch, keep=[b]) for b in bs]
        for k in range(3):
            for b in bs:
                b.hip.htod(np.full(b.q.size, 6.5, np.float32), b.out)
            for g in graphs[::-1 if k % 2 else 1]:
                g.launch()
            for b, w in zip(bs, want):
                np.testing.assert_array_equal(b.get(), w)
            bs[k].launch()
        for b, w in zip(bs, want):
            b.check(w)
        for g in graphs:
            g.close()
    finally:
        other.close()


# ---------------- refused calls ----------------
def test_refused_arguments(hip):
    b = hip.alloc(1 << 16)
    step = dict(nseq=4, q_start=b, parent=b, length=b, t=8, words=1, pos=b, mask=b)
    for bad in (dict(nseq=4097), dict(t=(1 << 24) + 1), dict(words=0), dict(words=9), dict(q_start=0), dict(parent=0), dict(length=0), dict(pos=0), dict(mask=0)):
        with pytest.raises(S.StrataError, match="tree_step"):
            hip.tree_step(**{**step, **bad})
    acc = dict(nseq=4, q_start=b, parent=b, tokens=b, ids=b, length=b, slots=b, t=8, words=1, max_path=4, n_path=b, chosen=b, last=b, keep=b, runs=b)
    for bad in (dict(nseq=4097), dict(t=(1 << 24) + 1), dict(words=0), dict(words=9), dict(max_path=0), dict(max_path=33), *(dict([(k, 0)]) for k in acc if acc[k] is b)):
        with pytest.raises(S.StrataError, match="tree_accept"):
            hip.tree_accept(**{**acc, **bad})
    fork = dict(nseq=4, src=0, keep=0, length=b, tables=b, max_pages=4, page=16, free=b, n_pages=8, n_free=b, refs=b, len_out=b, n_free_out=b, runs=b)
    for bad in (dict(nseq=4097), dict(page=8), dict(page=48), dict(n_pages=0), dict(n_pages=1 << 27), dict(max_pages=0), dict(nseq=4096, max_pages=1 << 19), dict(keep=b, len_out=b), dict(keep=b, runs=b, len_out=int(b) + 64),
                *(dict([(k, 0)]) for k in fork if fork[k] is b)):
        with pytest.raises(S.StrataError, match="kv_pages_fork"):
            hip.kv_pages_fork(**{**fork, **bad})
    move = dict(caches=b, n_caches=2, row_bytes=64, n_slots=8, runs=b, groups=2, per=3)
    for bad in (dict(row_bytes=0), dict(row_bytes=24), dict(row_bytes=(1 << 24) + 16), dict(per=0), dict(per=257), dict(n_slots=0), dict(n_slots=1 << 31), dict(groups=1 << 21), dict(groups=1 << 20, n_caches=1 << 11),
                dict(caches=0), dict(runs=0)):
        with pytest.raises(S.StrataError, match="kv_rows_move"):
            hip.kv_rows_move(**{**move, **bad})
    logp = dict(x=b, x_stride=64, n=64, rows=2, ids=b, m=1, logp=b, k=3, top_ids=b)
    for bad in (dict(n=0), dict(n=1 << 31), dict(rows=(1 << 20) + 1), dict(m=17), dict(k=65), dict(x=0), dict(x=int(b) + 2), dict(ids=0), dict(x_stride=63)):
        with pytest.raises(S.StrataError, match="logits_logprobs"):
            hip.logits_logprobs(**{**logp, **bad})
    attn = dict(q=b, kc=b, vc=b, qg=0, out=int(b) + 4096, t=4, max_q=4, pos=b, q_start=b, length=b, nseq=1, tables=b, max_pages=2, page=16, n_pages=4, nh=8, nkv=2, hd=64, scale=0.1, mask=b, words=1)
    for bad in (dict(mask=0), dict(words=0), dict(words=9), dict(win=31), dict(words=2, win=63), dict(hd=96), dict(nh=6), dict(page=8), dict(q=0), dict(kc=0), dict(vc=0), dict(out=0), dict(pos=0), dict(q_start=0), dict(length=0),
                dict(tables=0), dict(max_prefix=5), dict(t=(1 << 20) + 1), dict(max_q=0), dict(max_q=5), dict(q=int(b) + 4), dict(out=b), dict(scale=0.0), dict(scale=float("nan")), dict(nseq=4097)):
        with pytest.raises(S.StrataError, match="tree attention"):
            hip.attn_paged_tree(**{**attn, **bad})
