"""The operators that serve a batch of sequences over a paged KV cache, through the C ABI, against their plain restatements
(tests/serve_oracle.py): page steps and choices bit for bit, processed logits bit for bit in float32, q/k norms with rope
against the contiguous form's bits, attention against float64."""
import numpy as np
import pytest

import rustingstrata_amd as S
from tests import serve_oracle as V
from tests.helpers import normal, rel_l2

pytestmark = pytest.mark.gpu
GUARD = -77


def up(hip, a):
    return hip.upload(np.ascontiguousarray(a))


def i32(hip, v):
    return up(hip, np.asarray(v, dtype=np.int32).reshape(-1))


def get_i32(hip, b, n):
    return hip.get(b, np.int32, n)


# ---------------- page steps ----------------
class Step:
    """One kv_pages_step on the device; every output carries a guard word behind it."""

    def __init__(self, hip, add, length, tables, free, n_pages, n_free, page, max_pages, t_max, P=0, place=False):
        nseq = len(add)
        guard = lambda n: i32(hip, [GUARD] * (n + 1))  # noqa: E731
        self.hip, self.nseq, self.t_max, self.max_pages, self.n_pages = hip, nseq, t_max, max_pages, n_pages
        self.add, self.len, self.n_free = i32(hip, list(add) or [0]), i32(hip, list(length) or [0]), i32(hip, [n_free])
        self.tables, self.free = i32(hip, np.append(tables, GUARD)), i32(hip, np.append(free, GUARD))
        self.q_start, self.pos, self.slots = guard(nseq + 1), guard(t_max), guard(t_max)
        self.len_out, self.n_free_out = (self.len, self.n_free) if place else (guard(nseq), guard(1))
        self.err, self.P = i32(hip, [5]), i32(hip, [P])
        self.page = page

    def run(self):
        self.hip.kv_pages_step(self.nseq, self.add, self.len, self.tables, self.max_pages, self.page, self.free, self.n_pages,
                               self.n_free, self.t_max, self.q_start, self.pos, self.slots, self.len_out, self.n_free_out,
                               prefix_len=self.P, err=self.err)
        return self

    def check(self, want, place=False):
        for name, n in (("q_start", self.nseq + 1), ("pos", self.t_max), ("slots", self.t_max), ("len_out", self.nseq), ("n_free_out", 1),
                        ("tables", self.nseq * self.max_pages), ("free", self.n_pages)):
            got = get_i32(self.hip, getattr(self, name), n + (0 if place and name in ("len_out", "n_free_out") else 1))
            np.testing.assert_array_equal(got[:n], np.asarray(want[name]).reshape(-1), err_msg=name)
            assert len(got) == n or got[n] == GUARD, name
        assert get_i32(self.hip, self.err, 1)[0] == 5 + want["refused"]


def random_step(nseq, page, max_pages, t_max, seed, ends=0.1, wild=False):
    rng = np.random.default_rng(seed)
    length = rng.integers(0, max_pages * page - page // 2, nseq)
    add = np.where(rng.random(nseq) < 0.5, 1, rng.integers(0, max(2, 2 * t_max // max(nseq, 1)), nseq))
    add[rng.random(nseq) < ends] = -1
    if wild:  # lengths and counts outside their limits
        length[rng.random(nseq) < 0.2] = -3
        length[rng.random(nseq) < 0.1] = 2**31 - 1
        add[rng.random(nseq) < 0.1] = 2**31 - 1
        add[rng.random(nseq) < 0.1] = -2**31
    n_pages = int(nseq * max_pages + 3)
    order = rng.permutation(n_pages)
    tables = order[:nseq * max_pages].reshape(nseq, max_pages)
    free = np.concatenate([order[nseq * max_pages:], order])[:n_pages]
    return add.astype(np.int64), length, tables, free, n_pages


@pytest.mark.parametrize("nseq,page,max_pages,t_max,n_free,wild", [
    (1, 16, 1, 1, 3, False), (1, 64, 40, 3000, 60, False), (8, 64, 64, 8, 200, False), (63, 16, 9, 70, 40, False), (65, 128, 3, 4096, 30, False),
    (300, 16, 20, 4097, 900, False), (1000, 32, 5, 900, 17, False), (4096, 16, 4, 9000, 5000, False), (4095, 16, 2, 4000, 0, False),
    (200, 16, 7, 500, 100, True), (700, 32, 6, 5000, 4203, True)])
def test_pages_step(hip, nseq, page, max_pages, t_max, n_free, wild):
    """Every output, the tables and the stack, with refusals, in place as well as not, and the same again on the same inputs."""
    add, length, tables, free, n_pages = random_step(nseq, page, max_pages, t_max, seed=nseq + t_max, wild=wild)
    want = V.pages_step(add, length, tables, max_pages, page, free, n_pages, n_free, 1000, t_max)
    s = Step(hip, add, length, tables, free, n_pages, n_free, page, max_pages, t_max, P=1000)
    s.run().check(want)
    want["refused"] *= 2
    s.run().check(want)
    want["refused"] //= 2
    Step(hip, add, length, tables, free, n_pages, n_free, page, max_pages, t_max, P=1000, place=True).run().check(want, place=True)


def test_pages_step_of_nothing(hip):
    s = Step(hip, [], [], np.zeros(0, np.int64), np.arange(4), 4, 2, 16, 3, 5).run()
    s.check(dict(q_start=[0], pos=[-1] * 5, slots=[-1] * 5, len_out=[], n_free_out=[2], tables=[], free=range(4), refused=0))
    s = Step(hip, [0, 0], [0, 17], np.zeros(6, np.int64), np.arange(4), 4, -9, 16, 3, 0).run()
    s.check(dict(q_start=[0, 0, 0], pos=[], slots=[], len_out=[0, 17], n_free_out=[0], tables=[0] * 6, free=range(4), refused=0))


def test_pages_step_bad_pages(hip):
    """Page ids outside the pool: their slots are -1; a stack that would overflow keeps its first pages."""
    add, length = np.array([2, 20, -1]), np.array([3, 16, 40])
    tables, free = np.array([[-5, 0, 0], [9, 0, 0], [1, 2, 3]]), np.array([99, 0, 0, 0])
    want = V.pages_step(add, length, tables, 3, 16, free, 4, 2, 0, 40)
    assert want["refused"] == 1 and -1 in want["slots"][:22]
    Step(hip, add, length, tables, free, 4, 2, 16, 3, 40).run().check(want)


def test_pages_run_of_a_server(hip):
    """Random steps of 40 sequences with the state on the device, recorded once as a graph and replayed: lengths, tables and
    the stack follow the restatement, and every slot handed out belongs to one sequence."""
    rng = np.random.default_rng(3)
    nseq, page, max_pages, n_pages, t_max = 40, 16, 12, 200, 128
    length, tables, free, n_free = np.zeros(nseq, np.int64), np.zeros((nseq, max_pages), np.int64), rng.permutation(n_pages), n_pages
    s = Step(hip, np.zeros(nseq), length, tables, free, n_pages, n_free, page, max_pages, t_max, place=True)
    g = hip.record_graph(s.run, keep=[s])
    for k in range(60):
        add = np.where(rng.random(nseq) < 0.7, 1, rng.integers(0, 30, nseq))
        add[rng.random(nseq) < 0.08] = -1
        want = V.pages_step(add, length, tables, max_pages, page, free, n_pages, n_free, 0, t_max)
        hip.htod(add.astype(np.int32), s.add)
        hip.htod(np.array([5], np.int32), s.err)
        g.launch()
        s.check(want, place=True)
        length, tables, free, n_free = np.array(want["len_out"]), want["tables"], want["free"], want["n_free_out"]
        held = np.concatenate([tables[i, :-(-n // page)] for i, n in enumerate(length)] + [free[:n_free]])
        assert len(held) == len(set(held.tolist())) == n_pages
    g.close()


def test_pages_refused_arguments(hip):
    b = hip.alloc(65536)
    ok = dict(nseq=4, add=b, length=b, tables=b, max_pages=4, page=16, free=b, n_pages=8, n_free=b, t_max=8, q_start=b, pos=b, slots=b, len_out=b, n_free_out=b)
    for bad in (dict(nseq=4097), dict(page=8), dict(page=48), dict(page=1 << 17), dict(n_pages=0), dict(n_pages=1 << 27), dict(max_pages=0), dict(max_pages=1 << 27),
                dict(t_max=(1 << 24) + 1), dict(add=0), dict(length=0), dict(tables=0), dict(free=0), dict(n_free=0), dict(q_start=0), dict(pos=0), dict(slots=0),
                dict(len_out=0), dict(n_free_out=0)):
        with pytest.raises(S.StrataError, match="kv_pages_step"):
            hip.kv_pages_step(**{**ok, **bad})


# ---------------- logits ----------------
def logits_case(rows, n, hist, seed, bias=0, mask=False, special=False):
    rng = np.random.default_rng(seed)
    x = (4 * rng.standard_normal((rows, n))).astype(np.float32)
    if special:
        x[rng.random((rows, n)) < 0.2] = np.inf
        x[rng.random((rows, n)) < 0.1] = np.nan
        x[rng.random((rows, n)) < 0.2] = -np.inf
        x[rng.random((rows, n)) < 0.2] = np.finfo(np.float32).min
        x[rng.random((rows, n)) < 0.2] = -0.0
    h = rng.integers(-2, max(1, min(n + 2, 3 * hist)), (rows, hist)) if hist else np.zeros((rows, 1), np.int64)
    lens = rng.integers(0, hist + 3, rows) if hist else np.zeros(rows, np.int64)
    pen = np.stack([rng.uniform(0.8, 1.6, rows), rng.uniform(-0.5, 0.9, rows), rng.uniform(-0.5, 0.9, rows)], 1).astype(np.float32)
    b = [[(int(rng.integers(-1, n + 1)), float(np.float32(rng.normal(0, 3)))) for _ in range(rng.integers(0, bias + 1))] for _ in range(rows)]
    ok = rng.random((rows, n)) < rng.choice([0.01, 0.5, 1.0], (rows, 1)) if mask else None
    return x, h, lens, rng.integers(0, hist + 2, rows), pen, b, ok


def words(ok, pad=0):
    rows, n = ok.shape
    w = -(-n // 32)
    bits = np.ones((rows, (w + pad) * 32), bool)  # (bits past the row are set: they must not matter)
    bits[:, :n] = ok
    return np.packbits(bits, axis=1, bitorder="little").view(np.uint32)


def run_logits(hip, x, h, lens, first, last, pen, bias, ok, place=False, stride=0, pad=0, append=False):
    rows, n = x.shape
    stride = stride or n
    xs = np.full((rows, stride), 7.5, np.float32)
    xs[:, :n] = x
    xb = up(hip, xs)
    out = xb if place else up(hip, np.full((rows, stride + 3), 9.5, np.float32))
    os_ = stride if place else stride + 3
    hb, lb = i32(hip, h), i32(hip, lens)
    flat = [e for r in bias for e in r] if bias else []
    ids = i32(hip, [GUARD] * (rows + 1))
    kw = dict(hist=hb, hist_stride=h.shape[1], hist_len=lb, hist_from=i32(hip, first) if first is not None else 0, last=last, append=append)
    if pen is not None:
        kw["pen"] = up(hip, pen)
    if flat:
        kw.update(bias_start=i32(hip, np.cumsum([0] + [len(r) for r in bias])), bias_ids=i32(hip, [t for t, _ in flat]),
                  bias_vals=up(hip, np.array([v for _, v in flat], np.float32)), n_bias=len(flat))
    if ok is not None:
        kw.update(mask=up(hip, words(ok, pad)), mask_stride=-(-n // 32) + pad)
    hip.logits_process(xb, stride, out, os_, n, rows, ids=ids, **kw)
    got = hip.get(out, np.float32, rows * os_).reshape(rows, os_)
    assert (got[:, n:] == (7.5 if place else 9.5)).all()
    if not place:
        np.testing.assert_array_equal(hip.get(xb, np.uint32, xs.size), xs.view(np.uint32).reshape(-1))
    i = get_i32(hip, ids, rows + 1)
    assert i[rows] == GUARD
    return got[:, :n], i[:rows], get_i32(hip, hb, h.size).reshape(h.shape), get_i32(hip, lb, rows)


def same_bits(got, want):
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan)
    np.testing.assert_array_equal(got.view(np.uint32)[~nan], np.ascontiguousarray(want).view(np.uint32)[~nan])


@pytest.mark.parametrize("rows,n,hist,last,bias,mask", [
    (1, 1, 1, 0, 1, True), (3, 31, 5, 2, 3, True), (2, 32, 40, 0, 0, False), (5, 33, 0, 0, 2, True), (2, 4095, 3000, 0, 9, False), (3, 4096, 100, 64, 0, True),
    (4, 4097, 700, 0, 30, True), (7, 32003, 300, 64, 20, True), (2, 151936, 9000, 0, 300, True), (64, 1000, 64, 1, 5, False)])
@pytest.mark.parametrize("special", [False, True])
def test_logits_process(hip, rows, n, hist, last, bias, mask, special):
    """Every value and choice bit for bit (float32, one rounding a step), out of place, in place and with row strides."""
    x, h, lens, first, pen, b, ok = logits_case(rows, n, hist, seed=rows + n + hist, bias=bias, mask=mask, special=special)
    want, ids = V.logits_process(x, h, lens, first, last, pen, b, ok)
    for kw in (dict(), dict(place=True), dict(stride=n + 5, pad=2)):
        got, gi, _, _ = run_logits(hip, x, h, lens, first, last, pen, b, ok, **kw)
        same_bits(got, want)
        if not np.isnan(want[ok] if ok is not None else want).any():  # (which of two NaN is the greater goes by their bits)
            np.testing.assert_array_equal(gi, ids)


@pytest.mark.parametrize("rows,n,hist,last,bias,mask", [
    (4, 33, 5, 2, 3, True), (5, 4097, 700, 0, 30, True), (3, 8192, 100, 64, 0, True), (6, 32003, 300, 64, 20, False), (2, 151936, 9000, 0, 300, True), (64, 9000, 64, 1, 5, True)])
@pytest.mark.parametrize("nan", [False, True])
def test_logits_choices_among_special_values(hip, rows, n, hist, last, bias, mask, nan):
    """Every row's choice among infinities, zeros of both signs, the lowest value and, with nan, values that are not numbers: the
    greatest allowed one of the values that the call writes, by the total order of their bits, the first on ties; without nan
    that of the restatement."""
    x, h, lens, first, pen, b, ok = logits_case(rows, n, hist, seed=rows * n + nan, bias=bias, mask=mask, special=True)
    if not nan:
        x[np.isnan(x)] = 0.0
    x[0] = np.where(np.arange(n) % 3 == 0, np.float32(-0.0), -np.inf)
    x[1] = np.where(np.arange(n) % 5 == 2, np.finfo(np.float32).min, -np.inf)
    want, ids = V.logits_process(x, h, lens, first, last, pen, b, ok)
    allowed = ok if ok is not None else np.ones(x.shape, bool)
    for kw in (dict(), dict(place=True), dict(stride=n + 5, pad=2)):
        got, gi, _, _ = run_logits(hip, x, h, lens, first, last, pen, b, ok, **kw)
        same_bits(got, want)
        assert gi.tolist() == [V.argmax_total(np.ascontiguousarray(g), a) for g, a in zip(got, allowed)]
        rest = [r for r in range(rows) if not np.isnan(want[r][allowed[r]]).any()]
        assert (len(rest) == rows or nan) and gi[rest].tolist() == ids[rest].tolist()


def test_logits_parts_alone(hip):
    """Nothing asked: a copy and the argmax; each part by itself; a mask that leaves nothing, one, or only -inf."""
    x, h, lens, first, pen, b, ok = logits_case(4, 5000, 50, seed=1, bias=6, mask=True)
    ok[0], ok[1], ok[2] = False, False, False
    ok[1, 4999] = True
    ok[2, [17, 4500]] = True
    x[2, [17, 4500]] = -np.inf
    for p, bb, m in ((None, None, None), (pen, None, None), (None, b, None), (None, None, ok)):
        want, ids = V.logits_process(x, h, lens, first, 0, p, bb, m)
        got, gi, _, _ = run_logits(hip, x, h, lens, first, 0, p, bb, m)
        same_bits(got, want)
        np.testing.assert_array_equal(gi, ids)
    assert ids.tolist()[:3] == [-1, 4999, 17]


def test_logits_append_and_replay(hip):
    """append: the choice goes to the history's end while it has room, and a recorded step sees it when replayed."""
    rows, n, cap = 3, 6000, 12
    x = normal((rows, n), seed=5)
    hist, lens = np.zeros((rows, cap), np.int32), np.array([0, 5, 11], np.int32)
    pen = np.array([[1.5, 0.5, 0.25]] * rows, np.float32)
    ok = np.ones((rows, n), bool)
    xb, out, hb, lb, ids, pb = up(hip, x), hip.alloc(4 * x.size), up(hip, hist), up(hip, lens), hip.alloc(4 * rows), up(hip, pen)
    mb = up(hip, words(ok))

    def f():
        hip.logits_process(xb, n, out, n, n, rows, hist=hb, hist_stride=cap, hist_len=lb, pen=pb, mask=mb, mask_stride=-(-n // 32), ids=ids, append=True)

    hip.logits_process(xb, n, out, n, n, rows, ids=ids)  # (sizes the scratch)
    g = hip.record_graph(f, keep=[xb, out, hb, lb, ids, pb, mb])
    for k in range(8):
        want, wi = V.logits_process(x, hist, lens, None, 0, pen, None, ok)
        g.launch()
        same_bits(hip.get(out, np.float32, x.size).reshape(x.shape), want)
        np.testing.assert_array_equal(get_i32(hip, ids, rows), wi)
        for r in range(rows):
            if wi[r] >= 0 and lens[r] < cap:
                hist[r, lens[r]] = wi[r]
                lens[r] += 1
        np.testing.assert_array_equal(get_i32(hip, lb, rows), lens)
        np.testing.assert_array_equal(get_i32(hip, hb, rows * cap).reshape(rows, cap), hist)
        ok[0] = k != 3  # nothing allowed: nothing chosen, nothing appended
        hip.htod(words(ok), mb)
    g.close()


def test_logits_refused_arguments(hip):
    b = hip.alloc(4096)
    ok = dict(x=b, x_stride=100, out=b, out_stride=100, n=100, rows=2)
    for bad in (dict(n=0), dict(n=1 << 31), dict(rows=65536), dict(x=0), dict(out=0), dict(x_stride=99), dict(out_stride=99), dict(out_stride=101), dict(pen=b),
                dict(pen=b, hist=b), dict(pen=b, hist_len=b), dict(append=True, ids=b), dict(append=True, hist=b, hist_len=b), dict(mask=b, mask_stride=3),
                dict(bias_start=b, n_bias=1), dict(bias_start=b, n_bias=1, bias_ids=b), dict(hist_stride=1 << 31), dict(last=1 << 31), dict(n_bias=1 << 31)):
        with pytest.raises(S.StrataError, match="logits_process"):
            hip.logits_process(**{**ok, **bad})
    hip.logits_process(0, 0, 0, 0, 0, 0)  # no rows: nothing to do


def test_logits_of_the_longest_row(hip):
    """A row of 2^31 - 1 logits in place: the choice and its place in the history at its far end, the rest as it was."""
    n = 2**31 - 1
    x = hip.alloc(4 * n)
    hip.memset(x)
    for at, v in ((0, -1.0), (n // 2, 0.5), (n - 2, 2.0), (n - 1, 3.0)):
        hip.htod(np.array([v], np.float32), x, off=4 * at)
    h, lens, ids = i32(hip, [n - 1, n - 1, 0]), i32(hip, [2]), i32(hip, [GUARD, GUARD])
    hip.logits_process(x, n, x, n, n, 1, hist=h, hist_stride=3, hist_len=lens, pen=up(hip, np.array([[2.0, 0.25, 0.5]], np.float32)), ids=ids, append=True)
    assert get_i32(hip, ids, 2).tolist() == [n - 2, GUARD] and get_i32(hip, h, 3).tolist() == [n - 1, n - 1, n - 2] and get_i32(hip, lens, 1)[0] == 3
    for at, want in ((0, [-1.0, 0.0]), (n // 2 - 1, [0.0, 0.5, 0.0]), (n - 3, [0.0, 2.0, 3.0 / 2 - 0.25 * 2 - 0.5])):
        got = np.zeros(len(want), np.float32)
        hip.dtoh(x, 4 * at, got)
        assert got.tolist() == want


# ---------------- q/k norms and rope into pages ----------------
@pytest.mark.parametrize("t,nh,nkv,hd,n_rot", [(1, 32, 4, 128, 128), (5, 8, 8, 64, 64), (7, 4, 1, 96, 32), (16, 16, 2, 128, 128), (333, 32, 4, 128, 128), (700, 4, 4, 64, 32),
                                                 (3, 64, 8, 128, 128), (2, 40, 40, 64, 0), (9, 3, 2, 64, 64)])
def test_norm_rope_paged(hip, t, nh, nkv, hd, n_rot):
    """The bits of rms_norm_rope_qk_t where tokens sit at consecutive positions; at positions of their own within 2e-6 of
    float64 (an angle's sine is rounded once to float32, the norm sums in float32: at most hd + 6 roundings of 2^-24, on
    average their root); rows that are skipped or not stored leave everything as it was."""
    rng = np.random.default_rng(t)
    W, eps, base, n_slots = (nh + 2 * nkv) * hd, 1e-6, 1e6, t + 40
    qkv, qw, kw = normal((t, W), seed=t), 1 + 0.1 * normal(hd, seed=1), 1 + 0.1 * normal(hd, seed=2)
    slots = rng.permutation(n_slots)[:t]
    qb, qwb, kwb = up(hip, qkv), up(hip, qw), up(hip, kw)
    k0, v0 = int(qb) + 4 * nh * hd, int(qb) + 4 * (nh + nkv) * hd
    fill = np.full(n_slots * nkv * hd, 0x3C01, np.uint16)

    def run(pos, slots):
        qo, kc, vc = up(hip, np.full(t * nh * hd, 3.25, np.float32)), up(hip, fill), up(hip, fill)
        hip.rms_norm_rope_qk_paged(qb, W, hd, qwb, qo, nh, k0, W, kwb, nkv, hd, eps, n_rot, i32(hip, pos), base, v0, W, kc, vc, i32(hip, slots), n_slots, t)
        return (hip.get(qo, np.float32, t * nh * hd).reshape(t, nh, hd), *(hip.get(c, np.uint16, fill.size).reshape(n_slots, nkv, hd) for c in (kc, vc)))

    # consecutive positions: the contiguous form's bits
    p0 = 11
    qo, ko, kc, vc = hip.alloc(t * nh * hd * 4), hip.alloc(t * nkv * hd * 4), hip.alloc((t + p0) * nkv * hd * 2), hip.alloc((t + p0) * nkv * hd * 2)
    hip.rms_norm_rope_qk_t(qb, W, hd, qwb, qo, t * nh, nh, k0, W, kwb, ko, t * nkv, nkv, hd, eps, n_rot, i32(hip, [p0, 0]), base, v0, W, kc, vc)
    q, k, v = run(np.arange(p0, p0 + t), slots)
    np.testing.assert_array_equal(q.view(np.uint32).reshape(-1), hip.get(qo, np.uint32, t * nh * hd))
    for got, c in ((k, kc), (v, vc)):
        np.testing.assert_array_equal(got[slots], hip.get(c, np.uint16, (t + p0) * nkv * hd).reshape(-1, nkv, hd)[p0:])
        rest = np.delete(got, slots, axis=0)
        assert (rest == 0x3C01).all()
    # positions of their own, some rows skipped, some not stored
    pos = rng.integers(0, 1 << 20, t)
    pos[rng.random(t) < 0.2] = -1
    sl = slots.copy()
    sl[rng.random(t) < 0.2] = rng.choice([-1, -9, n_slots, 2**31 - 1])
    q, k, v = run(pos, sl)
    live = pos >= 0
    x = qkv.reshape(t, -1, hd).astype(np.float64)
    assert (q[~live] == 3.25).all()
    if live.any():
        want = V.norm_rope(x[live][:, :nh], qw.astype(np.float64), eps, n_rot, pos[live][:, None], base)
        assert np.abs(q[live] - want).max() <= 2e-6 * np.abs(want).max()
    stored = live & (sl >= 0) & (sl < n_slots)
    assert (np.delete(k, sl[stored], axis=0) == 0x3C01).all() and (np.delete(v, sl[stored], axis=0) == 0x3C01).all()
    if stored.any():
        want = V.norm_rope(x[stored][:, nh:nh + nkv], kw.astype(np.float64), eps, n_rot, pos[stored][:, None], base)
        # half a step of f16 (2^-11 relative, 2^-25 below the normal range) beyond the float32 error
        assert (np.abs(k[sl[stored]].view(np.float16) - want) <= 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + 2e-6 * np.abs(want).max()).all()
        np.testing.assert_array_equal(v[sl[stored]].view(np.float16), qkv.reshape(t, -1, hd)[stored][:, nh + nkv:].astype(np.float16))


def test_norm_rope_paged_refused_arguments(hip):
    b = hip.alloc(1 << 16)
    ok = dict(q=b, q_tstride=768, q_stride=64, qw=b, qo=b, qper=8, k=b, k_tstride=768, kw=b, kper=2, n=64, eps=1e-6, n_rot=64, pos=b, base=1e6, v=b, v_tstride=768,
              kc=b, vc=b, slots=b, n_slots=16, t=2)
    for bad in (dict(n=48), dict(n=0), dict(n=544), dict(n_rot=66), dict(n_rot=63), dict(qper=0), dict(kper=0), dict(q=0), dict(qw=0), dict(qo=0), dict(k=0), dict(kw=0),
                dict(pos=0), dict(v=0), dict(kc=0), dict(vc=0), dict(slots=0), dict(t=1 << 31), dict(t=1 << 28), dict(q_stride=63), dict(q_tstride=511), dict(k_tstride=127),
                dict(v_tstride=127)):
        with pytest.raises(S.StrataError, match="rms_norm_rope"):
            hip.rms_norm_rope_qk_paged(**{**ok, **bad})


# ---------------- attention ----------------
class Batch:
    """A batch over paged caches: q new rows and n cached keys a sequence, pages anywhere in the pool, the rest of the pool
    not a number (unused pages and the tails of used ones must not matter)."""

    def __init__(self, hip, q, n, nh, nkv, hd, page, P=0, seed=0, sink=False, gate=False, extra=0, big=False):
        rng = np.random.default_rng(seed)
        self.hip, self.nh, self.nkv, self.hd, self.page, self.P = hip, nh, nkv, hd, page, P
        self.qn, self.n, self.nseq = list(q), list(n), len(q)
        self.t = sum(q) + extra
        need = [-(-k // page) for k in n]
        pp = -(-P // page)
        self.max_pages, self.n_pages = max(need + [1]), sum(need) + pp + 3
        order = rng.permutation(self.n_pages)
        self.tables = rng.integers(-5, self.n_pages + 5, (self.nseq, self.max_pages))  # (entries past a sequence's pages: anything)
        at = 0
        self.kc, self.vc = (np.full((self.n_pages * page, nkv, hd), np.nan, np.float16) for _ in range(2))
        used = np.zeros(self.n_pages * page, bool)
        for s, k in enumerate(need):
            self.tables[s, :k] = order[at:at + k]
            j = np.arange(n[s])
            used[self.tables[s][j // page] * page + j % page] = True
            at += k
        self.prefix = order[at:at + max(pp, 1)]
        j = np.arange(P)
        used[self.prefix[j // page] * page + j % page] = True
        self.used = np.flatnonzero(used)
        self.kc[used] = rng.standard_normal((used.sum(), nkv, hd))
        self.vc[used] = 0.5 * rng.standard_normal((used.sum(), nkv, hd))
        self.q = (1.5 * rng.standard_normal((self.t, nh, hd))).astype(np.float32)
        if big:
            self.q[0] *= 20
        self.q_start = np.concatenate([[0], np.cumsum(q)])
        self.pos = np.concatenate([P + k - m + np.arange(m) for m, k in zip(q, n)] + [np.full(extra, 1 << 20)]).astype(np.int64)
        self.sink = rng.standard_normal(nh).astype(np.float32) if sink else None
        self.gate = rng.standard_normal((self.t, nh, 2, hd)).astype(np.float32) if gate else None
        self.scale = float(np.float32(1 / np.sqrt(hd)))
        self.max_q = max(q + [1])

    def upload(self):
        hip = self.hip
        self.b = dict(q=up(hip, self.q), kc=up(hip, self.kc), vc=up(hip, self.vc), qg=up(hip, self.gate) if self.gate is not None else 0,
                      pos=i32(hip, self.pos), q_start=i32(hip, self.q_start), length=i32(hip, self.n), tables=i32(hip, self.tables))
        self.pb = dict(prefix=i32(hip, self.prefix), prefix_len=i32(hip, [self.P]), sink=up(hip, self.sink) if self.sink is not None else 0)
        self.out = up(hip, np.full(self.q.size, 6.5, np.float32))
        return self

    def launch(self, win=0, max_prefix=None, max_q=None):
        mp = self.P if max_prefix is None else max_prefix
        p = dict(self.pb) if mp else dict(sink=self.pb["sink"])
        self.hip.attn_paged(out=self.out, t=self.t, max_q=max_q or self.max_q, nseq=self.nseq, max_pages=self.max_pages, page=self.page, n_pages=self.n_pages,
                            nh=self.nh, nkv=self.nkv, hd=self.hd, scale=self.scale, max_prefix=mp, win=win, **self.b, **p)

    def get(self):
        return self.hip.get(self.out, np.float32, self.q.size).reshape(self.q.shape)

    def want(self, win=0, rows=None):
        return V.attn(self.q, self.kc, self.vc, self.pos, self.q_start, self.n, self.tables, self.page, self.prefix, self.P, self.scale, win=win, sink=self.sink,
                      gate=self.gate[:, :, 1] if self.gate is not None else None, rows=rows)

    def check(self, got, win=0, rows=None):
        """Each row and head within 2^-23 (14 + max |s|) of its norm: a float32 score is off by 2^-24 |s| in its sum (of some
        hd / 8 steps, whose roundings mostly cancel) and again in the exponent, which is its weight's relative error; the exps, the splits (2^-22), the sums and the two joins of partial
        sums (an exp, a product and a sum each) add fourteen times 2^-23 at most."""
        want, top = self.want(win, rows if rows is None else set(rows))
        m = self.q_start[-1]
        assert (got[m:] == 6.5).all()
        for r in range(m) if rows is None else rows:
            for h in range(self.nh):
                w = want[r, h]
                assert np.isfinite(got[r, h]).all(), (r, h)
                if not w.any():
                    assert not got[r, h].any(), (r, h)
                else:
                    assert rel_l2(got[r, h], w) <= 2.0 ** -23 * (14 + top[r, h]), (r, h, rel_l2(got[r, h], w))


SHAPES = [(8, 1, 128), (8, 2, 64), (4, 2, 128), (4, 4, 64), (3, 3, 128)]


@pytest.mark.parametrize("nh,nkv,hd", SHAPES)
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("win", [0, 40])
def test_attn_paged_decode(hip, nh, nkv, hd, page, win):
    """One token a sequence, contexts of 0 to 1500 keys around the borders of pages and chunks; rows behind the last sequence."""
    n = [1, 0, 15, 16, 17, 63, 64, 65, 0, 128, 129, 255, 256, 257, 700, 1500, 2]
    b = Batch(hip, [1] * len(n), n, nh, nkv, hd, page, seed=nh + page, extra=2, big=True).upload()
    b.launch(win)
    b.check(b.get(), win)


@pytest.mark.parametrize("nh,nkv,hd", SHAPES)
@pytest.mark.parametrize("P,page", [(1, 16), (64, 64), (1000, 16), (2051, 128)])
@pytest.mark.parametrize("win", [0, 100])
def test_attn_paged_prefix(hip, nh, nkv, hd, P, page, win):
    """A shared prefix ahead of own keys, sequences without own keys among them, sinks and gates."""
    n = [5, 1, 200, 0, 64, 33, 1, 17, 90, 2]
    b = Batch(hip, [1] * len(n), n, nh, nkv, hd, page, P=P, seed=P, sink=P % 2 == 1, gate=P % 2 == 0, extra=1).upload()
    b.launch(win, max_prefix=P + 77)
    b.check(b.get(), win)


@pytest.mark.parametrize("nh,nkv,hd", SHAPES)
@pytest.mark.parametrize("q,n,P,win", [
    ([4, 1, 2, 3], [4, 300, 2, 65], 0, 0), ([3, 4, 1], [70, 4, 9], 130, 50), ([5, 1, 17, 0, 2], [5, 400, 200, 30, 2], 0, 0), ([40, 1, 33], [40, 90, 300], 65, 0),
    ([130, 1, 1, 70], [130, 513, 7, 470], 0, 90), ([300], [300], 0, 0), ([1, 129], [1, 129], 0, 0), ([200, 3], [200, 3], 700, 300)])
def test_attn_paged_ragged(hip, nh, nkv, hd, q, n, P, win):
    """Speculative tokens, prompt chunks from their start and with earlier context, decoding sequences among them; causal."""
    b = Batch(hip, q, n, nh, nkv, hd, 32, P=P, seed=len(q) + P, sink=P > 0, gate=win > 0, extra=3).upload()
    b.launch(win)
    b.check(b.get(), win)


def test_attn_paged_long(hip):
    """A context of 30000 keys beside short ones, and a prefix as long, on two head shapes; rows sampled."""
    for nh, nkv, hd in ((32, 4, 128), (8, 8, 64)):
        b = Batch(hip, [1, 1, 1], [30001, 5, 777], nh, nkv, hd, 64, seed=1).upload()
        b.launch()
        b.check(b.get())
        b = Batch(hip, [1, 2, 1], [3, 2, 100], nh, nkv, hd, 64, P=30011, seed=2).upload()
        b.launch()
        b.check(b.get())


@pytest.mark.parametrize("nh,nkv,hd,q,n,P,win", [
    (2, 2, 128, [300, 1, 40], [20000, 9000, 40], 0, 0), (2, 2, 64, [140, 260], [12000, 260], 4100, 0), (8, 1, 128, [100, 1, 1, 1, 90], [15000, 700, 1, 64, 90], 3001, 0),
    (8, 1, 64, [33, 1], [25000, 25000], 0, 9000), (4, 2, 128, [700], [700], 0, 0), (2, 1, 128, [9, 10, 8, 9], [3000, 10, 5000, 64], 0, 0)])
def test_attn_paged_deep_chunks(hip, nh, nkv, hd, q, n, P, win):
    """Prompt chunks deep in their contexts, whose tiles many blocks share, beside decoding sequences; rows at the borders of
    tiles and sequences."""
    b = Batch(hip, q, n, nh, nkv, hd, 64, P=P, seed=sum(q)).upload()
    b.launch(win)
    TT = 128 * nkv // nh
    rows = {r for s, m in zip(b.q_start, q) for r in [*range(s, s + m, TT), s + m - 1, s + m // 2, min(s + TT - 1, s + m - 1)]}
    b.check(b.get(), win, rows=sorted(rows)[:40])


@pytest.mark.parametrize("q,P", [([1] * 9, 0), ([1, 4, 2, 1], 70), ([60, 1, 17, 2, 33], 0), ([60, 1, 17, 2, 33], 130)])
@pytest.mark.parametrize("win", [0, 1, 37, 2**31 - 1])
def test_attn_paged_positions_in_any_order(hip, q, P, win):
    """Rows at any positions in any order: before the first key, past the last, twice the same; windows of one key and of all; a
    bound max_q of all rows."""
    rng = np.random.default_rng(win % 100 + P)
    n = rng.integers(0, 500, len(q)).tolist()
    b = Batch(hip, q, n, 8, 2, 64, 16, P=P, seed=P + 3, sink=True, gate=True)
    for s in range(len(q)):
        b.pos[b.q_start[s]:b.q_start[s + 1]] = rng.integers(-3, P + n[s] + 6, q[s])
    b.upload().launch(win, max_q=b.t)
    b.check(b.get(), win)


@pytest.mark.parametrize("nseq", [257, 1030, 4096])
@pytest.mark.parametrize("P", [0, 33])
def test_attn_paged_many_sequences(hip, nseq, P):
    """Hundreds to thousands of sequences: of no rows, decoding ones and short chunks, more tiles than a block plans at once."""
    rng = np.random.default_rng(nseq)
    q = rng.choice([0, 1, 2, 8, 9, 17], nseq, p=[0.1, 0.2, 0.1, 0.1, 0.3, 0.2])
    n = q + rng.integers(0, 40, nseq) * (rng.random(nseq) < 0.7)
    b = Batch(hip, q.tolist(), n.tolist(), 2, 1, 64, 16, P=P, seed=nseq, extra=5).upload()
    b.launch()
    rows = sorted({0, int(b.q_start[-1]) - 1} | set(rng.integers(0, b.q_start[-1], 400).tolist()))
    got = b.get()
    b.check(got, rows=rows)
    assert np.isfinite(got).all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("most", [1, 2, 4, 40])
@pytest.mark.parametrize("win,bad", [(0, False), (30, True)])
def test_attn_paged_rows_finished_in_one_launch(hip, hd, most, win, bad):
    """More (sequence, KV head) pairs than blocks: those that one block holds are finished there, others are joined; sinks, gates,
    sequences without keys or rows, and values that are not finite at keys that a sequence's earlier rows do not see."""
    rng = np.random.default_rng(most)
    nseq = 300
    q = rng.integers(0, min(most, 4) + 1, nseq)
    if most > 4:
        q[[7, 200]] = most
    n = np.where(rng.random(nseq) < 0.1, 0, q + rng.integers(0, 400, nseq))
    b = Batch(hip, q.tolist(), n.tolist(), 8, 2, hd, 16, seed=most, sink=True, gate=True, extra=2)
    rows = sorted(set(rng.integers(0, b.q_start[-1], 150).tolist()))
    want = b.want(win, set(rows))
    if bad:
        for s in range(nseq):
            if q[s] > 1 and n[s]:
                j = n[s] - 1
                b.vc[b.tables[s][j // 16] * 16 + j % 16] = np.inf
                rows = [r for r in rows if r != b.q_start[s + 1] - 1]
    b.want = lambda *a: want
    b.upload().launch(win)
    b.check(b.get(), win, rows=rows)


def test_attn_paged_two_graphs_of_one_context(hip):
    """Two recorded calls of one context share its workspace, which a larger eager call between them replaces."""
    a = Batch(hip, [1] * 4, [300, 3, 64, 900], 8, 2, 64, 16, P=70, seed=1).upload()
    c = Batch(hip, [60, 1, 3], [300, 80, 3], 8, 2, 64, 16, P=30, seed=2).upload()
    a.launch(), c.launch()
    wa, wc = a.get(), c.get()
    a.check(wa), c.check(wc)
    ga = hip.record_graph(a.launch, keep=[a])
    d = Batch(hip, [1] * 200, [100] * 200, 8, 8, 128, 16, P=300, seed=3).upload()
    d.launch()
    gc = hip.record_graph(c.launch, keep=[c])
    for _ in range(4):
        for b, g, w in ((a, ga, wa), (c, gc, wc)):
            hip.htod(np.full(b.q.size, 6.5, np.float32), b.out)
            g.launch()
            np.testing.assert_array_equal(b.get().view(np.uint32), w.view(np.uint32))
        d.launch()
    d.check(d.get(), rows=[0, 57, 199])
    ga.close(), gc.close()


def test_attn_paged_prefix_sums_of_decoding_rows_alone(hip):
    """Chunks of thousands of rows beside decoding sequences over a prefix: the context's scratch holds no sums of the prefix for the
    chunks' rows (134 MB here for each split of it), and the rows of either kind are right."""
    other = S.HipBackend(0)
    b = Batch(other, [1, 8189, 2], [40, 8189, 3], 32, 4, 128, 64, P=500, seed=11).upload()
    other.sync()
    before = other.mem_info()[0]
    b.launch()
    got = b.get()
    assert before - other.mem_info()[0] < 100 << 20  # (67 MB of cut tiles' sums, 4 of own keys', 6 of the prefix's)
    b.check(got, rows=[0, 1, 700, 8189, 8190, 8191])
    other.close()


def test_attn_paged_offsets_past_32_bits(hip):
    """A pool of 2.4 GB a cache whose used pages lie at its far end."""
    nh, nkv, hd, page = 16, 16, 128, 64
    b = Batch(hip, [1, 40], [100, 70], nh, nkv, hd, page, P=90, seed=4)
    far = 9400
    pool = [hip.alloc((far * page + len(b.kc)) * nkv * hd * 2) for _ in range(2)]
    assert far * page * nkv * hd * 2 > 1 << 31
    for p, c in zip(pool, (b.kc, b.vc)):
        hip.htod(c, p, off=far * page * nkv * hd * 2)
    b.upload()
    b.b.update(kc=pool[0], vc=pool[1], tables=i32(hip, b.tables + far))
    b.pb["prefix"] = i32(hip, b.prefix + far)
    b.n_pages += far
    b.launch()
    b.n_pages -= far
    b.check(b.get())


@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_attn_paged_non_finite(hip, bad):
    """A value that is not finite reaches the rows that see its key and no other: not rows of earlier positions in the same
    tile, not rows past a window, not other heads or sequences; a key that is not a number the rows that see it."""
    nh, nkv, hd, page = 8, 2, 64, 16
    for q, n, P, win in (([2, 1], [50, 60], 40, 0), ([2, 1], [50, 60], 40, 30), ([60, 1], [70, 60], 40, 0), ([60, 1], [70, 60], 40, 30)):
        b = Batch(hip, q, n, nh, nkv, hd, page, P=P, seed=6)
        clean, _ = b.want(win)
        for key in (n[0] - 1, 20, -1):  # the last own key of sequence 0, one in its middle, the prefix's last
            j = key if key >= 0 else P - 1
            slot = (b.tables[0] if key >= 0 else b.prefix)[j // page] * page + j % page
            at = P + key if key >= 0 else P - 1
            sees = (b.pos >= at) & ((b.pos - win < at) if win else True) & ((np.arange(b.t) < q[0]) if key >= 0 else True)
            for what in ("v", "k"):
                save = b.kc.copy(), b.vc.copy()
                (b.kc if what == "k" else b.vc)[slot, 1, 7] = np.nan if what == "k" else bad
                b.upload().launch(win)
                got = b.get()
                b.kc, b.vc = save
                hit = np.zeros(got.shape, bool)
                hit[np.ix_(sees, range(4, 8), range(hd) if what == "k" else [7])] = True
                assert not np.isfinite(got[hit]).any(), (q, key, what)
                ok = np.abs(got - clean)[~hit]
                assert np.isfinite(ok).all() and ok.max() <= 1e-5, (q, key, what)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("q,n,P,win", [([1, 1, 1, 2], [200, 1, 70, 33], 0, 0), ([1, 2, 1], [70, 40, 9], 130, 60), ([60, 1], [90, 50], 65, 0), ([4], [300], 0, 20)])
@pytest.mark.parametrize("size,scale", [(3e-35, None), (1e-36, None), (1e-38, None), (1e-44, None), (1.0, 1e-38), (1.0, 1e-45), (1e-38, 1e37)])
def test_attn_paged_tiny_queries(hip, hd, q, n, P, win, size, scale):
    """Queries down to the smallest float, in all heads of a row and in one, beside ordinary ones, and scales as small: the weights
    are those of scores near 0, not numbers that are not (decode rows, prefix and tiles; Batch.check's bound)."""
    b = Batch(hip, q, n, 8, 2, hd, 16, P=P, seed=sum(n), sink=True)
    if scale:
        b.scale = float(np.float32(scale))
        b.q *= np.float32(size)
    else:
        b.q[::2] *= np.float32(size)
        b.q[:, 5] *= np.float32(size)
    assert np.isfinite(b.q).all() and b.q[0].any()
    b.upload().launch(win)
    b.check(b.get(), win)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_attn_paged_non_finite_queries(hip, bad):
    """A query that is not finite spoils its own row of its head and no other bit: decode rows with and without a prefix, rows that a
    block finishes itself, tiles whole and cut."""
    for q, n, P in (([1, 2, 1], [300, 60, 5], 0), ([1, 2, 1], [300, 60, 5], 200), ([1] * 300, [20] * 300, 0), ([70, 1, 300], [900, 60, 300], 0), ([70, 1, 300], [900, 60, 300], 200)):
        b = Batch(hip, q, n, 8, 2, 64, 16, P=P, seed=P + len(q), sink=True).upload()
        b.launch()
        clean = b.get()
        for r, h in ((0, 3), (b.q_start[1] + q[1] - 1, 7), (b.t - 1, 0)):
            x = b.q.copy()
            x[r, h, 5] = bad
            hip.htod(x, b.b["q"])
            b.launch()
            got = b.get()
            assert not np.isfinite(got[r, h]).any(), (q[:3], P, r, h)
            got[r, h] = clean[r, h]
            np.testing.assert_array_equal(got.view(np.uint32), clean.view(np.uint32))


def test_attn_paged_holes(hip):
    """Page ids outside the pool hold no keys, in tables and prefix; a sequence of holes alone gives 0."""
    for q in ([1, 1, 1], [40, 3, 50]):
        n = [200, 90, 100]
        b = Batch(hip, q, n, 8, 2, 64, 16, P=100, seed=8)
        b.tables[0, [0, 3, 12]] = [-1, b.n_pages, 2**31 - 1]
        b.tables[1, :] = -1
        b.prefix[[1, 6]] = [-2**31, b.n_pages + 5]
        b.upload().launch()
        b.check(b.get())
        b.prefix[:] = -1
        b.upload().launch(win=60)
        got = b.get()
        b.check(got, win=60)
        assert not got[b.q_start[1]:b.q_start[2]].any()


def test_attn_paged_lengths_from_the_device(hip):
    """Lengths, tables and a prefix of 0 or more come from device memory: a recorded call replays with others; device lengths
    past the host's bounds are cut to them, and rows that max_q does not cover do not fault."""
    nh, nkv, hd, page = 8, 2, 64, 32
    b = Batch(hip, [1] * 6, [100, 1, 64, 300, 5, 31], nh, nkv, hd, page, P=200, seed=9).upload()
    b.launch()
    g = hip.record_graph(b.launch, keep=[b])
    for n, P in (([100, 1, 64, 300, 5, 31], 200), ([1, 1, 1, 1, 1, 1], 0), ([99, 0, 33, 257, 5, 2], 7), ([100, 1, 64, 300, 5, 31], 200)):
        b.n, b.P = n, P
        b.pos = np.array([P + k - 1 for k in n])
        hip.htod(np.array(n, np.int32), b.b["length"])
        hip.htod(b.pos.astype(np.int32), b.b["pos"])
        hip.htod(np.array([P], np.int32), b.pb["prefix_len"])
        g.launch()
        b.check(b.get())
    g.close()
    full = [b.max_pages * page] * 6
    hip.htod(np.array([2**31 - 1] * 6, np.int32), b.b["length"])
    hip.htod(np.array([2**31 - 1], np.int32), b.pb["prefix_len"])
    b.launch(max_prefix=200)
    b.n, b.P, b.used = full, 200, None
    assert b.get().shape == (6, nh, hd)
    b = Batch(hip, [40, 1], [40, 9], nh, nkv, hd, page, seed=1).upload()
    b.launch(max_q=1)
    b.check(b.get(), rows=[40])


@pytest.mark.parametrize("q,max_q", [([1] * 5, 1), ([1, 40, 1, 17, 2], 40)])
@pytest.mark.parametrize("win", [0, 50])
def test_attn_paged_device_lengths_past_their_bounds(hip, q, max_q, win):
    """Device lengths above max_pages pages and above max_prefix count as those, below 0 as 0."""
    page, pages, P = 32, 6, 90
    b = Batch(hip, q, [page * pages] * len(q), 8, 2, 64, page, P=P, seed=max_q + win, sink=True).upload()
    assert b.max_pages == pages
    for n, pl in ((2**31 - 1, 2**31 - 1), (page * pages + 1, P + 1), (-1, P), (-2**31, -2**31)):
        b.n, b.P = [min(max(n, 0), page * pages)] * len(q), min(max(pl, 0), P)
        hip.htod(np.array([n] * len(q), np.int32), b.b["length"])
        hip.htod(np.array([pl], np.int32), b.pb["prefix_len"])
        b.launch(win, max_prefix=P)
        got = b.get()
        b.check(got, win)
        assert got.any() == (n > 0 or (pl > 0 and not win))


def test_attn_paged_two_contexts(hip):
    """Calls of two contexts at once (streams of their own, workspaces of their own), captured and eager, give what one gives."""
    other = S.HipBackend(0)
    a = Batch(hip, [1] * 9, [500, 3, 900, 64, 65, 1, 2, 1200, 40], 8, 1, 128, 16, P=500, seed=1).upload()
    c = Batch(other, [1, 70, 2], [600, 200, 2], 8, 1, 128, 16, P=90, seed=2).upload()
    a.launch(), c.launch()
    wa, wc = a.get(), c.get()
    ga, gc = hip.record_graph(a.launch, keep=[a]), other.record_graph(c.launch, keep=[c])
    for _ in range(10):
        ga.launch(), gc.launch()
        c.launch(), a.launch()
    np.testing.assert_array_equal(a.get().view(np.uint32), wa.view(np.uint32))
    np.testing.assert_array_equal(c.get().view(np.uint32), wc.view(np.uint32))
    a.check(wa), c.check(wc)
    ga.close(), gc.close()
    other.close()


def test_attn_paged_matches_the_contiguous_forms(hip):
    """Consecutive pages are a contiguous cache: the same attention as attn_decode and attn_prefill (float32 sums in another
    order: twice the bound of either)."""
    nh, nkv, hd, page, n, t = 8, 2, 128, 64, 300, 50
    kc, vc, q = (normal((320, nkv, hd), seed=s).astype(np.float16) for s in (1, 2)), None, normal((t, nh, hd), seed=3)
    kc, vc = kc
    kb, vb, qb, out = up(hip, kc), up(hip, vc), up(hip, q), hip.alloc(q.size * 4)
    part = hip.alloc(4 * hip.attn_part_floats(nh, hd))
    tables = i32(hip, np.arange(5))
    s = 1 / np.sqrt(hd)
    for m in (1, t):
        if m == 1:
            hip.attn_decode(qb, kb, vb, 0, out, part, i32(hip, [n - 1, 0]), nh, nkv, hd, s, 1)
        else:
            hip.attn_prefill(qb, kb, vb, 0, out, i32(hip, [n - t, 0]), t, nh, nkv, hd, s)
        want = hip.get(out, np.float32, m * nh * hd).reshape(m, nh, hd)
        hip.attn_paged(qb, kb, vb, 0, out, m, m, i32(hip, np.arange(n - m, n)), i32(hip, [0, m]), i32(hip, [n]), 1, tables, 5, page, 5, nh, nkv, hd, s)
        got = hip.get(out, np.float32, m * nh * hd).reshape(m, nh, hd)
        for r in range(m):
            for h in range(nh):
                assert rel_l2(got[r, h], want[r, h]) <= 2.0 ** -22 * (14 + 6), (m, r, h)


def test_attn_paged_refused_arguments(hip):
    x, y = hip.alloc(1 << 16), hip.alloc(1 << 16)
    ok = dict(q=x, kc=x, vc=x, qg=0, out=y, t=2, max_q=1, pos=x, q_start=x, length=x, nseq=2, tables=x, max_pages=4, page=16, n_pages=8, nh=8, nkv=2, hd=64, scale=0.125)
    for bad in (dict(hd=96), dict(nh=6), dict(nh=32), dict(nkv=0), dict(nseq=4097), dict(page=24), dict(page=8), dict(n_pages=0), dict(n_pages=1 << 27), dict(max_pages=0),
                dict(max_pages=1 << 27), dict(q=0), dict(kc=0), dict(vc=0), dict(out=0), dict(pos=0), dict(q_start=0), dict(length=0), dict(tables=0), dict(max_q=0), dict(max_q=3),
                dict(t=(1 << 20) + 1), dict(max_prefix=5), dict(max_prefix=5, prefix=x), dict(max_prefix=5, prefix_len=x), dict(max_prefix=(1 << 30) + 1, prefix=x, prefix_len=x),
                dict(win=1 << 31), dict(q=int(x) + 4), dict(qg=int(x) + 4), dict(out=int(y) + 8), dict(out=x), dict(qg=y), dict(scale=0.0), dict(scale=-1.0), dict(scale=np.nan),
                dict(scale=np.inf), dict(kc=int(x) + 2), dict(vc=int(x) + 8), dict(nseq=4096, max_pages=1 << 26)):
        with pytest.raises(S.StrataError, match="paged attention"):
            hip.attn_paged(**{**ok, **bad})
    hip.attn_paged(**{**ok, "t": 0})
    hip.attn_paged(**{**ok, "nseq": 0})


def test_attn_paged_positions_up_to_31_bits(hip):
    """Bounds on a prefix and a sequence that pass 2^31 - 1024 positions together are refused; at that sum, a call whose device
    lengths are small is computed (a decoding row; a tile of rows)."""
    x, y = hip.alloc(1 << 16), hip.alloc(1 << 16)
    ok = dict(q=x, kc=x, vc=x, qg=0, out=y, t=1, max_q=1, pos=x, q_start=x, length=x, nseq=1, tables=x, max_pages=1 << 26, page=16, n_pages=8, nh=8, nkv=2, hd=64, scale=0.125,
              prefix=x, prefix_len=x)
    for P in (1 << 30, (1 << 30) - 1023):
        with pytest.raises(S.StrataError, match="positions of a prefix and a sequence"):
            hip.attn_paged(**{**ok, "max_prefix": P})
    for q in (1, 20):
        b = Batch(hip, [q], [50], 8, 2, 64, 16, P=70, seed=q, extra=1).upload()
        b.max_pages = 1 << 26
        b.launch(max_prefix=(1 << 30) - 1024)
        b.check(b.get())


# ---------------- the operators together ----------------
class Server:
    """A decode layer served with these operators: a step brings tokens of several sequences, whose q, k and v come from a table by
    token id; the attention's output row is its sequence's row of logits."""
    NH, NKV, HD, PAGE, NSEQ, MAX_PAGES, N_PAGES, T, CAP, P = 8, 2, 64, 16, 4, 6, 17, 70, 90, 21

    def __init__(self, hip, rng):
        self.hip, self.vocab = hip, self.NH * self.HD
        f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        self.tq, self.tk, self.tv = f(self.vocab, self.NH, self.HD), f(self.vocab, self.NKV, self.HD), f(self.vocab, self.NKV, self.HD)
        self.qw, self.kw = 1 + 0.1 * f(self.HD), 1 + 0.1 * f(self.HD)
        self.pre = rng.integers(0, self.vocab, self.P)
        kvd = self.NKV * self.HD
        self.kc, self.vc = (up(hip, np.full(self.N_PAGES * self.PAGE * kvd, np.nan, np.float16)) for _ in range(2))
        self.q, self.k, self.v = (hip.alloc(4 * self.T * n * self.HD) for n in (self.NH, self.NKV, self.NKV))
        self.qo, self.out = (hip.alloc(4 * self.T * self.vocab) for _ in range(2))
        self.qwb, self.kwb = up(hip, self.qw), up(hip, self.kw)
        self.tables = up(hip, np.full((self.NSEQ, self.MAX_PAGES), -1, np.int32))
        self.prefix = i32(hip, [self.N_PAGES - 1, self.N_PAGES - 2])  # the prefix on two pages that are never free
        self.free = i32(hip, rng.permutation(self.N_PAGES - 2))
        self.n_free, self.n_free0 = i32(hip, [self.N_PAGES - 2]), self.N_PAGES - 2
        self.add, self.len, self.err, self.plen = i32(hip, [0] * self.NSEQ), i32(hip, [0] * self.NSEQ), i32(hip, [0]), i32(hip, [0])
        self.q_start, self.pos, self.slots = (hip.alloc(4 * (self.T + 8)) for _ in range(3))
        self.hist, self.hlen, self.ids = hip.alloc(4 * self.NSEQ * self.CAP), i32(hip, [0] * self.NSEQ), i32(hip, [0] * self.NSEQ)
        self.pen = up(hip, np.tile(np.array([1.3, 0.2, 0.1], np.float32), (self.NSEQ, 1)))
        self.logits = hip.alloc(4 * self.NSEQ * self.vocab)

    def norm_rope(self, t, pos, slots):
        H = self.HD
        self.hip.rms_norm_rope_qk_paged(self.q, self.NH * H, H, self.qwb, self.qo, self.NH, self.k, self.NKV * H, self.kwb, self.NKV, H, 1e-6, H, pos, 1e4,
                                        self.v, self.NKV * H, self.kc, self.vc, slots, self.N_PAGES * self.PAGE, t)

    def inputs(self, tokens):
        for b, tab in ((self.q, self.tq), (self.k, self.tk), (self.v, self.tv)):
            self.hip.htod(np.ascontiguousarray(tab[tokens]), b)

    def cache_prefix(self):
        self.inputs(self.pre)
        pages = [self.N_PAGES - 1, self.N_PAGES - 2]
        self.norm_rope(self.P, i32(self.hip, np.arange(self.P)), i32(self.hip, [pages[i // self.PAGE] * self.PAGE + i % self.PAGE for i in range(self.P)]))
        self.hip.htod(np.array([self.P], np.int32), self.plen)

    def layer(self, t, max_q):
        self.hip.kv_pages_step(self.NSEQ, self.add, self.len, self.tables, self.MAX_PAGES, self.PAGE, self.free, self.N_PAGES, self.n_free, t, self.q_start,
                               self.pos, self.slots, self.len, self.n_free, prefix_len=self.plen, err=self.err)
        self.norm_rope(t, self.pos, self.slots)
        self.hip.attn_paged(self.qo, self.kc, self.vc, 0, self.out, t, max_q, self.pos, self.q_start, self.len, self.NSEQ, self.tables, self.MAX_PAGES, self.PAGE,
                            self.N_PAGES, self.NH, self.NKV, self.HD, self.HD ** -0.5, prefix=self.prefix, prefix_len=self.plen, max_prefix=2 * self.PAGE)

    def choose(self, x):
        self.hip.logits_process(x, self.vocab, self.logits, self.vocab, self.vocab, self.NSEQ, hist=self.hist, hist_stride=self.CAP, hist_len=self.hlen,
                                pen=self.pen, ids=self.ids, append=True)

    def check(self, toks, add):
        """The device's state after a layer against each sequence's tokens: keys and values at their slots, and the attention's rows
        from the cached values and roped queries in float64."""
        hip, H = self.hip, self.HD
        pool = lambda b: hip.get(b, np.float16, self.N_PAGES * self.PAGE * self.NKV * H).reshape(-1, self.NKV, H)  # noqa: E731
        kc, vc, tables = pool(self.kc), pool(self.vc), get_i32(hip, self.tables, self.NSEQ * self.MAX_PAGES).reshape(self.NSEQ, -1)
        prefix, length = get_i32(hip, self.prefix, 2), [len(x) for x in toks]
        for s, x in enumerate(toks):
            all_ = np.concatenate([self.pre, np.array(x, np.int64)]).astype(np.int64)
            got = [np.concatenate([V.rows_of(c, prefix, self.P, self.PAGE)[0], V.rows_of(c, tables[s], len(x), self.PAGE)[0]]) for c in (kc, vc)]
            np.testing.assert_array_equal(got[1], self.tv[all_].astype(np.float16))
            k = V.norm_rope(self.tk[all_].astype(np.float64), self.kw, 1e-6, H, np.arange(len(all_))[:, None], 1e4)
            # half a step of f16, and angles below 128 in float32 (their frequency's rounding, the product's, and sin and cos: 4 half
            # steps of 2^-24 times 128) turn a pair of values by 2^-15 of its length
            pair = np.hypot(k[..., :H // 2], k[..., H // 2:])
            assert (np.abs(got[0] - k) <= 2.0 ** -11 * np.abs(k) + 2.0 ** -15 * np.concatenate([pair, pair], -1) + 2.0 ** -25).all(), s
        rows = [max(a, 0) for a in add]
        q_start = np.concatenate([[0], np.cumsum(rows)])
        assert get_i32(hip, self.q_start, self.NSEQ + 1).tolist() == q_start.tolist()
        t = q_start[-1]
        qo, out = (hip.get(b, np.float32, self.T * self.vocab).reshape(self.T, self.NH, H)[:t] for b in (self.qo, self.out))
        pos = np.concatenate([self.P + n - m + np.arange(m) for n, m in zip(length, rows)])
        assert get_i32(hip, self.pos, t).tolist() == pos.tolist()
        want, top = V.attn(qo, kc, vc, pos, q_start, length, tables, self.PAGE, prefix, self.P, self.HD ** -0.5)
        for r in range(t):
            for h in range(self.NH):
                assert rel_l2(out[r, h], want[r, h]) <= 2.0 ** -23 * (14 + top[r, h]), (add, r, h)  # (Batch.check's bound)


def test_serving_a_batch(hip):
    """Prompts, chunks, decode steps, sequences that end and begin: every step's state and rows, pages back at the end."""
    rng = np.random.default_rng(5)
    sv = Server(hip, rng)
    sv.cache_prefix()
    toks = [[] for _ in range(sv.NSEQ)]  # cached tokens of each sequence
    # a step's new tokens a sequence (-1: it ends): prompts, a chunk beside decoding ones, decoding, an end, another's begin
    steps = [[20, 0, 3, 0], [1, 40, 1, 0], [1, 1, 1, 25], [1, 1, 1, 1], [1, 1, -1, 1], [1, 1, 0, 1], [1, 1, 17, 1]] + [[1, 1, 1, 1]] * 3 + [[-1, 1, 1, 1], [5, 1, 1, 1], [-1] * 4]
    for add in steps:
        new = [rng.integers(0, sv.vocab, max(a, 0)) for a in add]
        flat = np.concatenate(new).astype(np.int64)
        if len(flat):
            sv.inputs(flat)
        hip.htod(np.array(add, np.int32), sv.add)
        sv.layer(max(len(flat), 1), max(max(add), 1))
        for s, a in enumerate(add):
            toks[s] = [] if a < 0 else toks[s] + new[s].tolist()
        assert get_i32(hip, sv.len, sv.NSEQ).tolist() == [len(t) for t in toks]
        assert get_i32(hip, sv.n_free, 1)[0] == sv.n_free0 - sum(-(-len(t) // sv.PAGE) for t in toks)
        sv.check(toks, add)
    assert get_i32(hip, sv.err, 1)[0] == 0


def test_serving_steps_recorded(hip):
    """A recorded decode step (pages, keys and values, attention, choice, histories) replayed over page borders gives the bits of
    the same steps launched one by one."""
    runs = []
    for graph in (False, True):
        rng = np.random.default_rng(6)
        sv = Server(hip, rng)
        sv.cache_prefix()
        flat = rng.integers(0, sv.vocab, 35)
        sv.inputs(flat)
        hip.htod(np.array([16, 3, 15, 1], np.int32), sv.add)
        sv.layer(35, 16)
        sv.inputs(rng.integers(0, sv.vocab, sv.NSEQ))
        hip.htod(np.array([1] * sv.NSEQ, np.int32), sv.add)
        got = []

        def step():
            sv.layer(sv.NSEQ, 1)
            sv.choose(sv.out)

        if graph:
            save = [(b, hip.get(b, np.int32, n)) for b, n in ((sv.len, sv.NSEQ), (sv.n_free, 1), (sv.hlen, sv.NSEQ))]
            step()  # (sizes the workspace)
            for b, x in save:
                hip.htod(x, b)
            g = hip.record_graph(step, keep=[sv])
        for k in range(40):
            g.launch() if graph else step()
            got.append((hip.get(sv.logits, np.uint32, sv.NSEQ * sv.vocab), get_i32(hip, sv.ids, sv.NSEQ), get_i32(hip, sv.len, sv.NSEQ)))
        runs.append(got)
        assert get_i32(hip, sv.err, 1)[0] == 0
        assert get_i32(hip, sv.len, sv.NSEQ).tolist() == [56, 43, 55, 41]
        if graph:
            g.close()
    for k, (a, b) in enumerate(zip(*runs)):
        for x, y in zip(a, b):
            np.testing.assert_array_equal(x, y, err_msg=str(k))
    assert len({tuple(i) for _, i, _ in runs[0]}) > 3  # (the penalties move the choices)


class Loop:
    """The steps of a server around one Server, as they are documented: each sequence's history is its prompt and what it has
    chosen, a step's new tokens are the history's next ones, and a sequence chooses with the row of its history's last token.
    Rows of the others are masked; a refused sequence's choice is taken back."""

    def __init__(self, hip, seed):
        self.hip, self.rng = hip, np.random.default_rng(seed)
        self.sv = sv = Server(hip, self.rng)
        sv.cache_prefix()
        self.rows, self.mask = up(hip, np.zeros((sv.NSEQ, sv.vocab), np.float32)), hip.alloc(sv.NSEQ * sv.vocab // 8)
        self.cached, self.hist = [0] * sv.NSEQ, [[] for _ in range(sv.NSEQ)]
        self.pen, self.err, self.refusals = np.tile(np.array([1.3, 0.2, 0.1], np.float32), (sv.NSEQ, 1)), 0, 0

    def begin(self, s, n):
        self.hist[s] = self.rng.integers(0, self.sv.vocab, n).tolist()
        self.hip.htod(np.array(self.hist[s], np.int32), self.sv.hist, off=4 * s * self.sv.CAP)
        self.hip.htod(np.array([n], np.int32), self.sv.hlen, off=4 * s)

    def step(self, add, graph=None):
        """add[s] > 0 (or 0 to wait, -1 to end). graph: a recorded step of one token of each sequence. Returns who was refused."""
        hip, sv, n = self.hip, self.sv, self.sv.NSEQ
        new = [h[c:c + max(a, 0)] for h, c, a in zip(self.hist, self.cached, add)]
        assert [len(x) for x in new] == [max(a, 0) for a in add]
        chooses = np.array([a > 0 and c + a == len(h) for h, c, a in zip(self.hist, self.cached, add)])
        lens, hist = np.array([len(h) for h in self.hist]), np.zeros((n, sv.CAP), np.int64)
        for s, h in enumerate(self.hist):
            hist[s, :len(h)] = h
        if any(new):
            sv.inputs(np.concatenate(new).astype(np.int64))
        hip.htod(np.array(add, np.int32), sv.add)
        ok = np.repeat(chooses[:, None], sv.vocab, 1)
        if graph:
            graph.launch()
            rows = hip.get(sv.out, np.float32, n * sv.vocab).reshape(n, -1)
        else:
            sv.layer(max(sum(map(len, new)), 1), max(max(add), 1))
            for s, end in enumerate(np.cumsum([len(x) for x in new])):
                if chooses[s]:
                    hip.dtod(sv.out, 4 * sv.vocab * int(end - 1), self.rows, 4 * sv.vocab * s, 4 * sv.vocab)
            hip.htod(words(ok), self.mask)
            hip.logits_process(self.rows, sv.vocab, sv.logits, sv.vocab, sv.vocab, n, hist=sv.hist, hist_stride=sv.CAP, hist_len=sv.hlen, pen=sv.pen,
                               mask=self.mask, mask_stride=sv.vocab // 32, ids=sv.ids, append=True)
            rows = hip.get(self.rows, np.float32, n * sv.vocab).reshape(n, -1)
        ids, length = get_i32(hip, sv.ids, n), get_i32(hip, sv.len, n)
        y, want = V.logits_process(rows, hist, lens, None, 0, self.pen, None, ok)
        same_bits(hip.get(sv.logits, np.float32, n * sv.vocab).reshape(n, -1), y)
        np.testing.assert_array_equal(ids, want)
        assert (ids[~chooses] == -1).all() and np.isfinite(rows).all()
        refused = [s for s, a in enumerate(add) if a > 0 and length[s] == self.cached[s]]
        for s, a in enumerate(add):
            if a < 0:
                self.cached[s] = 0
                self.begin(s, 0)
            elif s in refused:
                hip.htod(np.array([len(self.hist[s])], np.int32), sv.hlen, off=4 * s)
            else:
                self.cached[s] += a
                self.hist[s] += [int(ids[s])] if chooses[s] else []
        err = get_i32(hip, sv.err, 1)[0]
        assert err - self.err == len(refused)
        self.err, self.refusals = err, self.refusals + len(refused)
        # cached lengths and histories have not parted: lengths, tokens, and the cached rows of the histories' tokens
        assert get_i32(hip, sv.len, n).tolist() == self.cached
        assert get_i32(hip, sv.hlen, n).tolist() == [len(h) for h in self.hist]
        device = get_i32(hip, sv.hist, n * sv.CAP).reshape(n, sv.CAP)
        for s, h in enumerate(self.hist):
            assert device[s, :len(h)].tolist() == h, s
        if not refused:
            sv.check([h[:c] for h, c in zip(self.hist, self.cached)], add)
        return refused


def test_serving_mixed_steps(hip):
    """Steps in which some sequences decode, some wait, end or bring a part of a prompt, and one finds no room: only the sequences
    whose last token is in get another, and the refused one's step can be made again."""
    lp = Loop(hip, 7)
    lp.begin(0, 20), lp.begin(1, 50), lp.begin(2, 3)
    for add in ([20, 30, 3, 0], [1, 20, 0, 0], [0, 0, 1, 0], [1, 1, 1, 0]):
        assert not lp.step(add)
    assert [len(h) for h in lp.hist] == [23, 52, 6, 0]
    lp.begin(3, 60)
    for add in ([0, 0, 0, 59], [1, 1, 1, 1]):
        assert not lp.step(add)
    for _ in range(5):  # (sequence 3 takes its fifth page)
        assert not lp.step([0, 1, 0, 1])
    assert not lp.step([1, 0, -1, 0])
    lp.begin(2, 66)
    for _ in range(2):
        assert lp.step([1, 1, 66, 0]) == [2]
    assert lp.hist[2] and len(lp.hist[2]) == 66
    assert not lp.step([0, -1, 0, 0])
    assert not lp.step([1, 0, 66, 1])
    assert len(lp.hist[2]) == 67 and lp.refusals == 2
    assert not lp.step([-1, 0, -1, -1])
    assert get_i32(hip, lp.sv.n_free, 1)[0] == lp.sv.n_free0


def test_serving_recorded_steps_refused(hip):
    """A recorded decode step replayed until sequences find no room, whose choices are taken back until another's end makes room:
    tokens as if nothing had been refused."""
    lp = Loop(hip, 8)
    for s, n in enumerate((50, 30, 62, 45)):
        lp.begin(s, n)
    assert not lp.step([50, 0, 0, 0]) and not lp.step([0, 30, 0, 0]) and not lp.step([0, 0, 62, 0]) and not lp.step([0, 0, 0, 45])

    def step():
        lp.sv.layer(lp.sv.NSEQ, 1)
        lp.sv.choose(lp.sv.out)

    g = hip.record_graph(step, keep=[lp])
    refused = [lp.step([1] * 4, graph=g) for _ in range(7)]
    assert refused == [[]] * 3 + [[3]] * 4
    assert not lp.step([-1, 0, 0, 0])
    lp.begin(0, 4)
    assert not lp.step([4, 0, 0, 0])
    for _ in range(5):
        assert not lp.step([1] * 4, graph=g)
    assert lp.refusals == 4 and [len(h) for h in lp.hist] == [lp.cached[s] + 1 for s in range(4)]
    g.close()


def test_serving_cached_keys(hip):
    """The cached keys after prompts and decode steps: float64 within half a step of f16 (2^-11 of the value, 2^-25 below the normal
    range) and the float32 arithmetic of a rope pair: 64 roundings of the sum of squares, halved by the root, the root's, the
    inverse's and two products' 4, and 3 each for the two terms of a turn whose sine and cosine are rounded once from double:
    48 times 2^-24 of the pair's length."""
    lp, H = Loop(hip, 9), Server.HD
    sv = lp.sv
    lp.begin(0, 30), lp.begin(2, 36)
    for add in ([30, 0, 20, 0], [1, 0, 16, 0], [1, 0, 1, 0], [1, 0, 1, 0]):
        assert not lp.step(add)
    kc = hip.get(sv.kc, np.float16, sv.N_PAGES * sv.PAGE * sv.NKV * H).reshape(-1, sv.NKV, H)
    tables, prefix = get_i32(hip, sv.tables, sv.NSEQ * sv.MAX_PAGES).reshape(sv.NSEQ, -1), get_i32(hip, sv.prefix, 2)
    for rows, toks, p0 in ((V.rows_of(kc, prefix, sv.P, sv.PAGE)[0], sv.pre, 0), *((V.rows_of(kc, tables[s], lp.cached[s], sv.PAGE)[0], lp.hist[s][:lp.cached[s]], sv.P) for s in (0, 2))):
        k = V.norm_rope(sv.tk[np.array(toks)].astype(np.float64), sv.kw.astype(np.float64), 1e-6, H, p0 + np.arange(len(toks))[:, None], 1e4)
        pair = np.hypot(k[..., :H // 2], k[..., H // 2:])
        f32 = 48 * 2.0 ** -24 * np.concatenate([pair, pair], -1)
        assert len(rows) and (np.abs(rows - k) <= (2.0 ** -11 * np.abs(k) + 2.0 ** -25 + f32) * (1 + 2.0 ** -10)).all()
