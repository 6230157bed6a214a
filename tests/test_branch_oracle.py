"""The plain restatements of the operators for drafted trees and branching sequences against known answers (CPU)."""
import numpy as np
import pytest

from tests import branch_oracle as B
from tests import serve_oracle as V

# 0 - 1 - 3 - 5, 0 - 2 - 4: a tree of six
TREE = [-1, 0, 0, 1, 2, 3]


def test_tree_known_answers():
    pos, mask, bad = B.tree_step([0, 6, 7], TREE + [-1], [16, 1], 100, 9, 1)
    assert pos.tolist() == [110, 111, 111, 112, 112, 113, 100, -1, -1] and bad == 0
    assert mask[:, 0].tolist() == [1, 3, 5, 11, 21, 43, 1, 0, 0]
    # parents that are not below their rows are roots; more rows than bits are a line
    pos, mask, bad = B.tree_step([0, 3], [0, 5, -2], [3], -4, 3, 1)
    assert bad == 3 and pos.tolist() == [0, 0, 0] and mask[:, 0].tolist() == [1, 2, 4]
    pos, mask, _ = B.tree_step([0, 40], [0] * 40, [50], 0, 40, 1)
    assert pos.tolist() == list(range(10, 50)) and not mask.any()


def test_accept_known_answers():
    tokens, slots = [9, 7, 8, 5, 6, 4], [32, 33, 34, 35, 36, 37]
    d = B.tree_accept([0, 6], TREE, tokens, [8, 0, 6, 0, 3, 0], [16], slots, 1, 4)
    # the path 0, 2, 4: choices 8, 6, 3
    assert d["n_path"] == [3] and d["chosen"].tolist() == [[8, 6, 3, -1]] and d["last"] == [4] and d["keep"] == [13]
    assert d["runs"].tolist() == [[[0, 0, 0], [34, 33, 1], [36, 34, 1], [0, 0, 0]]]
    d = B.tree_accept([0, 6], TREE, tokens, [8, 0, 6, 0, 3, 0], [16], slots, 1, 2)
    assert d["n_path"] == [2] and d["keep"] == [12]
    d = B.tree_accept([0, 0, 2], [-1, 0], [1, 2], [2, 3], [5, 7], [-1, 4], 1, 2)
    assert d["n_path"].tolist() == [0, 0] and d["keep"].tolist() == [5, 7] and d["last"].tolist() == [-1, -1]


def fork(src, keep, length, tables, free, refs, n_pages=12, page=16, max_pages=4):
    f = np.array(list(free) + [0] * (n_pages - len(free)))
    return B.pages_fork(src, keep, np.array(length), np.array(tables), max_pages, page, f, n_pages, len(free), np.array(refs))


def test_fork_known_answers():
    # sequence 1 goes on from 0: page 1 shared, page 2 copied to 9; its own page 3 goes back
    d = fork([0, 0], None, [24, 5], [[1, 2, 0, 0], [3, 0, 0, 0]], [8, 9], [0] * 12)
    assert d["tables"].tolist() == [[1, 2, 0, 0], [1, 9, 0, 0]] and d["refs"][1] == 1 and d["refs"].sum() == 1
    assert d["runs"].tolist() == [[0, 0, 0], [32, 144, 8]] and d["n_free_out"] == [2] and d["free"][:2].tolist() == [8, 3] and d["len_out"].tolist() == [24, 24]
    # two that change places hand their pages over
    d = fork([1, 0], None, [24, 5], [[1, 2, 0, 0], [3, 0, 0, 0]], [], [0] * 12)
    assert d["tables"][0, 0] == 3 and d["tables"][1, :2].tolist() == [1, 2] and not d["refs"].any() and not d["runs"].any() and d["len_out"].tolist() == [5, 24]
    # a cut into a page that another holds takes a copy; a cut into one's own does not
    d = fork(None, [20, 30], [40, 40], [[1, 2, 3, 0], [1, 2, 4, 0]], [7], [0, 1, 1] + [0] * 9)
    assert d["refused"] == 1 and d["tables"].tolist() == [[1, 7, 3, 0], [1, 2, 4, 0]] and d["len_out"].tolist() == [20, 40]
    assert d["refs"][:3].tolist() == [0, 1, 0] and d["free"][0] == 3 and d["n_free_out"] == [1]
    d = fork(None, [20], [40], [[1, 2, 3, 0]], [], [0] * 12)
    assert d["len_out"] == [20] and d["free"][0] == 3 and d["n_free_out"] == [1]
    # ended, and so no heir but itself; no such source; no page for one that was to become another
    d = fork([0, 5, 0], [0, 3, 3], [40, 20, 17], [[1, 2, 3, 0], [4, 5, 0, 0], [6, 8, 0, 0]], [], [0] * 12)
    assert d["refused"] == 2 and d["len_out"].tolist() == [0, 20, 0] and d["free"][:5].tolist() == [1, 2, 3, 6, 8] and d["n_free_out"] == [5]
    d = fork([0, 0], [16, 24], [24, 5], [[1, 2, 0, 0], [3, 0, 0, 0]], [], [0] * 12)
    assert d["refused"] == 1 and d["len_out"].tolist() == [16, 0] and d["free"][:2].tolist() == [2, 3]


def test_random_forks_keep_the_pool_whole():
    """After any run of forks, cuts, ends and steps every page is on the stack or held by as many sequences as refs says, and a
    page that a sequence may still write is held by it alone; what a sequence reads is what it should."""
    rng = np.random.default_rng(0)
    nseq, page, max_pages, n_pages = 7, 16, 5, 30
    length, tables, free, n_free, refs = np.zeros(nseq, np.int64), np.zeros((nseq, max_pages), np.int64), rng.permutation(n_pages), n_pages, np.zeros(n_pages, np.int64)
    cache, text, mark = np.zeros(n_pages * page, np.int64), [[] for _ in range(nseq)], 0
    for k in range(300):
        src = rng.integers(0, nseq, nseq) if k % 3 else None
        keep = rng.integers(0, max_pages * page, nseq) if k % 2 else None
        d = B.pages_fork(src, keep, length, tables, max_pages, page, free, n_pages, n_free, refs)
        new = []
        for s in range(nseq):
            u = s if src is None else src[s]
            want = text[u] if keep is None else text[u][:keep[s]]
            new.append(want if d["len_out"][s] == len(want) else text[s] if u == s else [])
        B.rows_move(cache, d["runs"][:, None], n_pages * page)
        length, tables, free, n_free, refs, text = d["len_out"], d["tables"], d["free"], d["n_free_out"][0], d["refs"], new
        add = rng.integers(0, 12, nseq)
        d = V.pages_step(add, length, tables, max_pages, page, free, n_pages, n_free, 0, 200)
        for s in range(nseq):
            for i in range(d["q_start"][s], d["q_start"][s + 1]):
                if d["slots"][i] >= 0:
                    mark += 1
                    cache[d["slots"][i]] = mark
                    text[s] = text[s] + [mark]
        length, tables, free, n_free = np.array(d["len_out"]), d["tables"], d["free"], d["n_free_out"]
        held = np.bincount(np.concatenate([tables[s, :-(-n // page)] for s, n in enumerate(length)] + [free[:n_free]]).astype(int), minlength=n_pages)
        np.testing.assert_array_equal(held, refs + 1)
        for s, n in enumerate(length):
            j = np.arange(n)
            assert cache[tables[s, j // page] * page + j % page].tolist() == text[s], (k, s)
            if n % page:
                assert refs[tables[s, n // page]] == 0


def test_logprobs_known_answers():
    x = np.log(np.array([[1, 2, 4, 1, 0]], np.float32) + 0.0, where=np.array([[1, 1, 1, 1, 0]], bool), out=np.full((1, 5), -np.inf, np.float32))
    logp, rank, h, ids, top = B.logprobs(x, np.array([[3, 1, 4, 9, -1]]), 6)
    assert np.allclose(np.exp(logp[0, :2]), [1 / 8, 1 / 4]) and np.isneginf(logp[0, 2:]).all() and rank.tolist() == [[4, 2, 5, 0, 0]]
    assert ids.tolist() == [[2, 1, 0, 3, 4, -1]] and np.allclose(np.exp(top[0]), [0.5, 0.25, 0.125, 0.125, 0, 0])
    assert np.isclose(h[0], 0.5 * np.log(2) + 0.25 * np.log(4) + 0.25 * np.log(8))


@pytest.mark.parametrize("P", [0, 5])
def test_attention_of_a_line_is_the_line_s(P):
    """A tree without branches, and a line of more rows than bits, see what attention by position shows them."""
    rng = np.random.default_rng(1)
    for n, length in ((6, 20), (40, 45)):
        q = rng.standard_normal((n, 2, 64)).astype(np.float32)
        kc, vc = (rng.standard_normal((96, 1, 64)).astype(np.float16) for _ in range(2))
        tables, prefix = np.array([[3, 1, 5]]), np.array([4])
        pos, mask, _ = B.tree_step([0, n], [i - 1 for i in range(n)], [length], P, n, 1)
        for win in (0, 33):
            got, _ = B.attn_tree(q, kc, vc, pos, mask, [0, n], [length], tables, 16, prefix, P, 0.1, 1, win=win)
            want, _ = V.attn(q, kc, vc, pos, [0, n], [length], tables, 16, prefix, P, 0.1, win=win)
            np.testing.assert_array_equal(got, want)
