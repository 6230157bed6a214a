"""Plain restatements of the operators for drafted trees and branching sequences (numpy): positions, masks, paths and page tables
with Python lists, rows moved one after the other, log probabilities and attention in float64."""
import numpy as np

from tests import serve_oracle as V


def tree_step(q_start, parent, length, P, t, words):
    """pos, mask [t, words] and the number of parents that are not below their rows."""
    pos, mask, bad = np.full(t, -1, np.int64), np.zeros((t, words), np.uint32), 0
    for s in range(len(length)):
        q0 = min(max(q_start[s], 0), t)
        n = min(max(q_start[s + 1], q0), t) - q0
        first = max(P, 0) + max(int(length[s]) - n, 0)
        for i in range(n):
            r = q0 + i
            if n > 32 * words:
                pos[r] = min(first + i, 2**31 - 1)
                continue
            p = int(parent[r])
            if p < -1 or p >= i:
                bad += 1
                p = -1
            if p >= 0:
                mask[r] = mask[q0 + p]
            mask[r, i // 32] |= np.uint32(1 << (i % 32))
            pos[r] = min(first + sum(int(w).bit_count() if hasattr(int, "bit_count") else bin(int(w)).count("1") for w in mask[r]) - 1, 2**31 - 1)
    return pos, mask, bad


def tree_accept(q_start, parent, tokens, ids, length, slots, words, max_path):
    B, t = len(length), len(parent)
    n_path, last, keep = np.zeros(B, np.int64), np.full(B, -1, np.int64), np.array(length, np.int64)
    chosen, runs = np.full((B, max_path), -1, np.int64), np.zeros((B, max_path, 3), np.int64)
    for s in range(B):
        q0 = min(max(q_start[s], 0), t)
        n = min(max(q_start[s + 1], q0), t) - q0
        if n == 0 or slots[q0] < 0:
            continue
        if n > 32 * words:
            n_path[s], last[s], chosen[s, 0] = 1, q0 + n - 1, ids[q0 + n - 1]
            continue
        path = [0]
        while len(path) < max_path and ids[q0 + path[-1]] >= 0:
            kids = [i for i in range(path[-1] + 1, n) if parent[q0 + i] == path[-1] and tokens[q0 + i] == ids[q0 + path[-1]]]
            if not kids:
                break
            path.append(kids[0])
        for i, r in enumerate(path):
            chosen[s, i] = ids[q0 + r]
            if r != i:
                runs[s, i] = slots[q0 + r], slots[q0 + i], 1
        n_path[s], last[s], keep[s] = len(path), q0 + path[-1], max(int(length[s]) - n, 0) + len(path)
    return dict(n_path=n_path, chosen=chosen, last=last, keep=keep, runs=runs)


def pages_fork(src, keep, length, tables, max_pages, page, free, n_pages, n_free, refs):
    """What kv_pages_fork leaves: tables, free, refs, len_out, n_free_out, runs, refused."""
    B, limit = len(length), max_pages * page
    old, tables, free, refs0 = tables, tables.copy(), free.copy(), refs
    held = [min(max(int(n), 0), limit) for n in length]
    top, refused = min(max(int(n_free), 0), n_pages), 0
    ok = [src is None or 0 <= src[s] < B for s in range(B)]
    u = [int(src[s]) if src is not None and ok[s] else s for s in range(B)]
    k = [min(max(int(keep[s]), 0), held[u[s]]) if keep is not None and ok[s] else held[u[s]] for s in range(B)]
    kids = {v: [s for s in range(B) if u[s] == v] for v in set(u)}
    heir = {v: v if v in ks else ks[0] for v, ks in kids.items()}
    most = {v: max(k[s] // page for s in ks) for v, ks in kids.items()}
    pool = lambda p: 0 <= p < n_pages  # noqa: E731
    count, out, runs, drop = refs.astype(np.int64).copy(), np.array(length, np.int64), np.zeros((B, 3), np.int64), []
    for s in range(B):
        refused += not ok[s]
        full, rem, other = k[s] // page, k[s] % page, u[s] != s
        if not other and k[s] == held[s]:
            continue
        take = copy = False
        if rem:
            pg = int(old[u[s], full])
            take = not pool(pg) or (heir[u[s]] == s and most[u[s]] <= full and refs0[pg] == 0)
            copy = not take
        if copy and top == 0:
            refused += 1
            if not other:
                continue
            full, copy, k[s] = 0, False, 0
        out[s] = k[s]
        mine = full + take  # pages from the old table of u
        if other:
            tables[s, :mine] = old[u[s], :mine]
            for p in old[u[s], :mine]:
                if pool(p):
                    count[p] += 1
        if copy:
            top -= 1
            fresh = int(free[top])
            tables[s, full] = fresh
            if pool(fresh):
                runs[s] = pg * page, fresh * page, rem
        drop += [int(p) for p in old[s, 0 if other else mine:-(-held[s] // page)]]
    for p in drop:
        if pool(p):
            count[p] -= 1
    lost = False
    for p in drop:
        if pool(p) and count[p] < 0:
            count[p] = 0
            if top < n_pages:
                free[top] = p
                top += 1
            else:
                lost = True
    return dict(tables=tables, free=free, refs=count, len_out=out, n_free_out=[top], runs=runs, refused=refused + lost)


def rows_move(cache, runs, n_slots):
    """cache [slots, ..] after the runs [groups, per, 3], in order."""
    for group in runs:
        for a, b, n in group:
            if n > 0 and a >= 0 and b >= 0 and a + n <= n_slots and b + n <= n_slots:
                for i in range(n):
                    cache[b + i] = cache[a + i]
    return cache


def order_key(x):
    """Unsigned keys in the order of strata_argmax_rows: larger is greater."""
    b = x.view(np.int32).astype(np.int64)
    return np.where(b < 0, -(b & 0x7FFFFFFF) - 1, b)


def logprobs(x, ids, k):
    """logp [rows, m], rank, entropy, top_ids [rows, k], top_logp of rows of float32 logits, in float64."""
    rows, n = x.shape
    m = ids.shape[1]
    logp, rank, entropy = np.full((rows, m), -np.inf), np.zeros((rows, m), np.int64), np.zeros(rows)
    top_ids, top_logp = np.full((rows, k), -1, np.int64), np.full((rows, k), -np.inf)
    for r in range(rows):
        v = x[r].astype(np.float64)
        with np.errstate(all="ignore"):
            if np.isneginf(v).all():
                y = np.full(n, -np.inf)
            elif np.isnan(v).any() or np.isposinf(v).any():
                y, entropy[r] = np.full(n, np.nan), np.nan
            else:
                y = v - v.max()
                p = np.exp(y)
                ls, entropy[r] = np.log(p.sum()), np.log(p.sum()) - (p[p > 0] * y[p > 0]).sum() / p.sum()
                y = y - ls
        order = np.argsort(-order_key(x[r]), kind="stable")
        place = np.empty(n, np.int64)
        place[order] = np.arange(n)
        for i, v in enumerate(ids[r]):
            if 0 <= v < n:
                logp[r, i], rank[r, i] = y[v], place[v] + 1
        c = min(k, n)
        top_ids[r, :c], top_logp[r, :c] = order[:c], y[order[:c]]
    return logp, rank, entropy, top_ids, top_logp


def attn_tree(q, kc, vc, pos, mask, q_start, length, tables, page, prefix, P, scale, words, win=0, sink=None, gate=None, rows=None):
    """serve_oracle.attn with ancestor masks [t, words]: out, and each row and head's largest score magnitude."""
    t, nh, hd = q.shape
    nkv = kc.shape[1]
    out, top = np.full((t, nh, hd), np.nan), np.zeros((t, nh))
    pk, pok = V.rows_of(kc, prefix, P, page)
    pv, _ = V.rows_of(vc, prefix, P, page)
    for s in range(len(length)):
        n, q0, q1 = int(length[s]), q_start[s], q_start[s + 1]
        k, ok = V.rows_of(kc, tables[s], n, page)
        v, _ = V.rows_of(vc, tables[s], n, page)
        k, v, ok = np.concatenate([pk, k]), np.concatenate([pv, v]), np.concatenate([pok, ok])
        at, base = np.arange(P + n), max(n - (q1 - q0), 0)
        for r in range(q0, q1):
            if rows is not None and r not in rows:
                continue
            if q1 - q0 > 32 * words:
                see = ok & (at <= pos[r])
            else:
                j = at - P - base  # which of the rows a key is
                bit = np.zeros(P + n, bool)
                mine = (j >= 0) & (j <= r - q0)
                bit[mine] = (mask[r, j[mine] // 32] >> (j[mine] % 32).astype(np.uint32)) & 1
                see = ok & ((j < 0) | bit)
            see = see & ((at > pos[r] - win) if win else True)
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
