"""Plain restatements of the batch-serving operators (numpy): page steps with Python lists, processed logits in float32 one
rounding a step, attention over pages and q/k norms with rope in float64."""
import numpy as np


def pages_step(add, length, tables, max_pages, page, free, n_pages, n_free, P, t_max):
    """What kv_pages_step leaves: q_start, pos, slots, len_out, n_free_out, tables, free, refused."""
    tables, free, P = tables.copy(), free.copy(), max(P, 0)
    limit = max_pages * page
    stack = list(free[:min(max(n_free, 0), n_pages)])
    refused, lost = 0, False
    for a, n, row in zip(add, length, tables):
        if a < 0 and n > 0:
            for pg in row[:-(-min(n, limit) // page)]:
                if len(stack) < n_pages:
                    stack.append(pg)
                else:
                    lost = True
    free[:len(stack)] = stack
    q_start, pos, slots, length_out = [0], [], [], []
    start = want = 0
    empty = len(stack)  # pages that the sequences so far leave
    left = empty
    for a, n, row in zip(add, length, tables):
        take = max(a, 0)
        need = 0
        bad = take > 0 and (n < 0 or n + take > limit or start + take > t_max)
        if take and not bad:
            need = -(-(n + take) // page) - -(-n // page)
            want += need
            bad = need > 0 and want > empty
        for i in range(max(n, 0), max(n, 0) + take):
            if len(pos) == t_max:
                break
            slot = -1
            if not bad:
                if i // page >= -(-n // page) and (i % page == 0):
                    row[i // page] = free[left - 1]
                    left -= 1
                pg = row[i // page]
                slot = pg * page + i % page if 0 <= pg < n_pages else -1
            pos.append(min(P + i, 2**31 - 1))  # (positions are int32, cut at its largest)
            slots.append(slot)
        start += take
        q_start.append(min(start, t_max))
        refused += bad
        length_out.append(0 if a < 0 else n if bad else n + take)
    pad = [-1] * (t_max - len(pos))
    return dict(q_start=q_start, pos=pos + pad, slots=slots + pad, len_out=length_out, n_free_out=left, tables=tables, free=free,
                refused=refused + lost)


def argmax_total(y, ok):
    """The greatest allowed value under the total order of floats, the first on ties; -1 if none is allowed."""
    b = y.view(np.int32).astype(np.int64)
    key = np.where(b < 0, -(b & 0x7FFFFFFF) - 1, b)
    key = np.where(ok, key, np.int64(-1) << 40)
    return int(np.argmax(key)) if ok.any() else -1


def logits_process(x, hist, hist_len, hist_from, last, pen, bias, ok):
    """x [rows, n] float32; bias: per row a list of (token, value); ok [rows, n] booleans. Returns y, ids."""
    y, ids = x.astype(np.float32).copy(), []
    n = x.shape[1]
    for r in range(x.shape[0]):
        with np.errstate(all="ignore"):
            if pen is not None:
                end = min(max(int(hist_len[r]), 0), hist.shape[1])
                lo = max(end - last, 0) if last else 0
                h = hist[r, lo:end]
                at = np.arange(lo, end)
                inside = (h >= 0) & (h < n)
                rep, freq, pres = pen[r].astype(np.float32)
                seen = np.unique(h[inside])
                y[r, seen] = np.where(y[r, seen] > 0, y[r, seen] / rep, y[r, seen] * rep)
                tok, cnt = np.unique(h[inside & (at >= (hist_from[r] if hist_from is not None else 0))], return_counts=True)
                y[r, tok] = (y[r, tok] - freq * cnt.astype(np.float32)) - pres
            for t, b in dict(bias[r] if bias else []).items():
                if 0 <= t < n:
                    y[r, t] = y[r, t] + np.float32(b)
        allowed = ok[r] if ok is not None else np.ones(n, bool)
        y[r, ~allowed] = -np.inf
        ids.append(argmax_total(y[r], allowed))
    return y, np.array(ids, dtype=np.int32)


def norm_rope(x, w, eps, n_rot, pos, base):
    """x [.., n] float64 heads, pos broadcast over them."""
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    half = n_rot // 2
    a = np.asarray(pos, dtype=np.float64)[..., None] * np.float64(np.float32(base)) ** (-2.0 * np.arange(half) / n_rot)
    c, s = np.cos(a), np.sin(a)
    p, q = y[..., :half].copy(), y[..., half:n_rot].copy()
    y[..., :half], y[..., half:n_rot] = p * c - q * s, p * s + q * c
    return y


def rows_of(pool, table, n, page):
    """The cached rows of positions 0 .. n - 1, and whether their page exists."""
    j = np.arange(n)
    pg = table[j // page] if n else np.zeros(0, np.int64)
    ok = (pg >= 0) & (pg < len(pool) // page)
    return pool[np.where(ok, pg, 0) * page + j % page].astype(np.float64), ok


def attn(q, kc, vc, pos, q_start, length, tables, page, prefix, P, scale, win=0, sink=None, gate=None, rows=None):
    """q [t, nh, hd]; kc, vc [slots, nkv, hd]. Returns out (rows from q_start[-1] on NaN) and each row and head's largest
    score magnitude (of the keys it sees). rows: only these (the others NaN)."""
    t, nh, hd = q.shape
    nkv = kc.shape[1]
    out, top = np.full((t, nh, hd), np.nan), np.zeros((t, nh))
    pk, pok = rows_of(kc, prefix, P, page)
    pv, _ = rows_of(vc, prefix, P, page)
    for s in range(len(length)):
        n = int(length[s])
        k, ok = rows_of(kc, tables[s], n, page)
        v, _ = rows_of(vc, tables[s], n, page)
        k, v, ok = np.concatenate([pk, k]), np.concatenate([pv, v]), np.concatenate([pok, ok])
        at = np.arange(P + n)
        for r in range(q_start[s], q_start[s + 1]):
            if rows is not None and r not in rows:
                continue
            see = ok & (at <= pos[r]) & ((at > pos[r] - win) if win else True)
            for h in range(nh):
                g = h // (nh // nkv)
                sc = k[see][:, g] @ q[r, h].astype(np.float64) * scale
                m = max([*sc[:0], sc.max() if len(sc) else -np.inf, sink[h] if sink is not None else -np.inf])
                e = np.exp(sc - m) if len(sc) else sc
                den = e.sum() + (np.exp(sink[h] - m) if sink is not None else 0.0)
                out[r, h] = e @ v[see][:, g] / den if len(sc) else 0.0
                top[r, h] = np.abs(sc).max() if len(sc) else 0.0
    if gate is not None:
        out *= 1.0 / (1.0 + np.exp(-gate.astype(np.float64)))
    return out, top
