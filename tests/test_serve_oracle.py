"""The plain restatements of the batch-serving operators against known answers (CPU)."""
import numpy as np

from tests import serve_oracle as V


def step(add, length, tables, free, n_pages=8, page=16, max_pages=4, t_max=64, P=0):
    return V.pages_step(add, length, np.array(tables), max_pages, page, np.array(list(free) + [0] * (n_pages - len(free))), n_pages, len(free), P, t_max)


def test_pages_known_answers():
    # sequence 0 fills its page, sequence 1 ends (its page 5 goes on the stack and comes off first), sequence 2 opens two
    d = step([1, -1, 17], [15, 3, 16], [[2, 0, 0, 0], [5, 0, 0, 0], [1, 0, 0, 0]], [7, 6], P=100)
    assert d["q_start"] == [0, 1, 1, 18] and d["len_out"] == [16, 0, 33] and d["n_free_out"] == 1 and d["refused"] == 0
    assert d["slots"][0] == 2 * 16 + 15 and d["slots"][1] == 5 * 16 and d["slots"][16] == 5 * 16 + 15 and d["slots"][17] == 6 * 16
    assert d["pos"][:3] == [115, 116, 117] and d["pos"][18:] == [-1] * 46 and d["tables"][2].tolist() == [1, 5, 6, 0]


def test_pages_refusals():
    # too few pages for sequence 0; sequence 1 then finds none either, sequence 2 needs none
    d = step([40, 1, 1], [0, 16, 3], [[0] * 4, [4, 0, 0, 0], [3, 0, 0, 0]], [7, 6])
    assert d["refused"] == 2 and d["len_out"] == [0, 16, 4] and d["n_free_out"] == 2
    assert d["slots"][:41] == [-1] * 41 and d["slots"][41] == 3 * 16 + 3
    # past max_pages; past t_max (rows cut); negative length
    d = step([65, 3, 60], [0, -1, 0], [[0] * 4] * 3, [7, 6, 5, 4, 3], t_max=100)
    assert d["refused"] == 3 and d["q_start"] == [0, 65, 68, 100] and d["slots"] == [-1] * 100


def test_logits_known_answers():
    x = np.array([[2.0, -2.0, 1.0, 4.0, 0.0]], np.float32)
    hist = np.array([[0, 1, 1, 9, -3, 3]], np.int32)
    y, ids = V.logits_process(x, hist, [6], [2], 0, np.array([[2.0, 0.5, 0.25]]), [[(2, 1.0), (2, 7.0), (8, 1.0)]], np.array([[1, 1, 1, 0, 1]], bool))
    # 0: before index 2, repetition alone; 1: repetition, counted once from index 2 on; 2: the last bias; 3: not allowed
    assert y.tolist() == [[1.0, -4.0 - 0.5 - 0.25, 8.0, -np.inf, 0.0]] and ids.tolist() == [2]
    y, ids = V.logits_process(x, hist, [6], None, 1, np.array([[2.0, 0.5, 0.25]]), None, np.zeros((1, 5), bool))
    assert np.isneginf(y).all() and ids.tolist() == [-1]
    z = np.array([-0.0, 0.0, np.nan, 1.0], np.float32)
    assert V.argmax_total(z, np.ones(4, bool)) == 2 and V.argmax_total(z, np.array([1, 1, 0, 0], bool)) == 1


def test_attention_known_answers():
    hd = 64
    q = np.ones((2, 2, hd), np.float32)
    kc, vc = np.zeros((64, 1, hd), np.float16), np.zeros((64, 1, hd), np.float16)
    vc[:, 0, 0] = np.arange(64)
    # equal scores: the mean of the rows seen; the prefix on page 3, the own keys on page 1
    out, _ = V.attn(q, kc, vc, [17, 4], [0, 2], [2], np.array([[1]]), 16, np.array([3]), 16, 1.0)
    assert np.isclose(out[0, 0, 0], (sum(range(48, 64)) + 16 + 17) / 18) and np.isclose(out[1, 1, 0], 50.0)
    out, _ = V.attn(q, kc, vc, [17, 4], [0, 2], [2], np.array([[1]]), 16, np.array([-1]), 16, 1.0, win=2, sink=np.zeros(2))
    assert np.isclose(out[0, 0, 0], 33 / 3) and (out[1] == 0).all()
