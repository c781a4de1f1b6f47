"""Plain restatements, in numpy float64 and Python integers, of the operators on the paged cache (include/qk_kernels.h:
qkk_attn_prep_axes, qkk_attn_packed, qkk_attn_tree, qkk_kv_resize, qkk_kv_fork, qkk_kv_compact).
TEST INFRASTRUCTURE ONLY: imported by tests/; the product never imports it.  Parity with another engine is unpinned:
the reference has no such operators; tests/test_kv_oracle.py pins these by what the definitions fix."""
import numpy as np


class Cache:
    """k, v [layer][page][kv head][row][dh]; table [seq][page] (None: sequence s is page s); ref, length lists of ints."""

    def __init__(self, k, v, table, ref=None, length=None):
        self.k, self.v, self.table = k, v, table
        self.ref, self.length = ref, length
        self.page_rows, self.n_page = k.shape[3], k.shape[1]
        self.n_seq = len(table) if table is not None else k.shape[1]
        self.cap = self.page_rows * (len(table[0]) if table is not None else 1)

    def at(self, seq, r):
        """(page, row in it) of cache row r, or None."""
        if r >= self.cap:
            return None
        page = seq if self.table is None else int(self.table[seq][r // self.page_rows])
        return (page, r % self.page_rows if self.table is not None else r) if 0 <= page < self.n_page else None


def runs(n_rows, start, seq, pos, cache, max_run):
    """(row, sequence, cache row, first row of the run, index in the run) of every row that is in a run in range."""
    for i, (s, p) in enumerate(zip(seq, pos)):
        if not (0 <= s < cache.n_seq and 0 <= p <= cache.cap):
            continue
        for r in range(start[i], min(start[i + 1], start[i] + max_run)):
            yield r, s, p + r - start[i], start[i], r - start[i]


def rope_axes(sections, in_turn):
    if not in_turn:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, out = list(sections), []
    while sum(left):
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                out.append(a)
    return out


def prep_axes(cache, layer, rows, q, kin, vin, qn, kn, rope, axis, axis_pos, dh, eps):
    """Writes k and v of the cache (their dtype); returns qhat float64, NaN where no run has the row."""
    half = rope.shape[1]
    out = np.full((q.shape[0], q.shape[1], dh), np.nan)

    def turned(x, w, row):
        x = x.astype(np.float64)
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
        p = np.clip([axis_pos[a][row] for a in axis], 0, rope.shape[0] - 1)
        c, s = (rope[p, np.arange(half), i].astype(np.float64) for i in (0, 1))
        y = x.copy()
        y[:, :half] = x[:, :half] * c - x[:, half:2 * half] * s
        y[:, half:2 * half] = x[:, :half] * s + x[:, half:2 * half] * c
        return y

    for row, seq, at, _, _ in rows:
        out[row] = turned(q[row][:, :dh], qn, row)
        place = cache.at(seq, at)
        if place is not None:
            cache.k[layer, place[0], :, place[1]] = turned(kin[row], kn, row).astype(cache.k.dtype)
            cache.v[layer, place[0], :, place[1]] = vin[row].astype(cache.v.dtype)
    return out


def attend(cache, layer, rows, q, gate=None, parent=None):
    """att float64 [rows][hQ][dh], NaN where no run has the row; parent None: packed, else a tree."""
    hq, dh = q.shape[1:]
    hkv = cache.k.shape[2]
    att = np.full(q.shape, np.nan)
    for row, seq, at, r0, node in rows:
        pos = at - node
        if parent is None:
            sees = list(range(at + 1))
        else:
            kin, a = [], node
            while True:
                kin.append(a)
                up = int(parent[r0 + a])
                if not 0 <= up < a:
                    break
                a = up
            sees = list(range(pos)) + [pos + a for a in sorted(kin)]
        places = [x for x in (cache.at(seq, r) for r in sees) if x is not None]
        if not places:
            att[row] = 0.0
        else:
            pages, inside = (np.array([p[i] for p in places]) for i in (0, 1))
            K, V = (x[layer, pages, :, inside].astype(np.float64) for x in (cache.k, cache.v))  # [keys][hkv][dh]
            for h in range(hq):
                g = h // (hq // hkv)
                sc = K[:, g] @ q[row, h].astype(np.float64) / np.sqrt(float(dh))
                e = np.exp(sc - sc.max())
                att[row, h] = e @ V[:, g] / e.sum()
        if gate is not None:
            att[row] = att[row] / (1 + np.exp(-gate[row, :, dh:].astype(np.float64)))
    return att


def resize(cache, new):
    """One sequence after the other; returns the status."""
    n = cache.page_rows
    if any(x > cache.cap for x in new):
        return -1
    if cache.table is None:
        cache.length = [x if x >= 0 else o for x, o in zip(new, cache.length)]
        return 0
    pages = lambda rows: -(-rows // n)  # noqa: E731
    for s, x in enumerate(new):
        if 0 <= x < cache.length[s]:
            for b in range(pages(x), pages(cache.length[s])):
                cache.ref[cache.table[s][b]] -= 1
                cache.table[s][b] = -1
            cache.length[s] = x
    free = [p for p, r in enumerate(cache.ref) if r == 0]
    shared = [r > 1 for r in cache.ref]
    grow = [(s, x) for s, x in enumerate(new) if x > cache.length[s]]
    split = {s: cache.length[s] % n and shared[cache.table[s][cache.length[s] // n]] for s, _ in grow}
    need = sum(pages(x) - pages(cache.length[s]) + bool(split[s]) for s, x in grow)
    if need > len(free):
        return need - len(free)
    for s, x in grow:
        old = cache.length[s]
        if split[s]:
            was, p = cache.table[s][old // n], free.pop(0)
            for pool in (cache.k, cache.v):
                pool[:, p, :, :old % n] = pool[:, was, :, :old % n]
            cache.ref[was] -= 1
            cache.ref[p] = 1
            cache.table[s][old // n] = p
        for b in range(pages(old), pages(x)):
            cache.table[s][b] = free.pop(0)
            cache.ref[cache.table[s][b]] = 1
        cache.length[s] = x
    return 0


def fork(cache, src, dst):
    if any(not (0 <= a < cache.n_seq and 0 <= b < cache.n_seq) or cache.length[b] for a, b in zip(src, dst)) or len(set(dst)) < len(dst):
        return -1
    was = list(cache.length)
    for a, b in zip(src, dst):
        cache.length[b] = was[a]
        if cache.table is None:
            for pool in (cache.k, cache.v):
                pool[:, b, :, :was[a]] = pool[:, a, :, :was[a]]
        else:
            for i in range(-(-was[a] // cache.page_rows)):
                cache.table[b][i] = cache.table[a][i]
                cache.ref[cache.table[a][i]] += 1
    return 0


def compact(cache, seq, base, path, n_path):
    for s, b, p, n in zip(seq, base, path, n_path):
        p = list(p[:max(n, 0)])
        if not 0 <= s < cache.n_seq or b < 0 or n < 1 or n > len(path[0]) or p != sorted(set(p)) or p[0] < 0:
            continue
        places = [(cache.at(s, b + a), cache.at(s, b + j)) for j, a in enumerate(p)]
        if any(x is None for pair in places for x in pair):
            continue
        for pool in (cache.k, cache.v):
            rows = [pool[:, f[0], :, f[1]].copy() for f, _ in places]
            for (_, to), r in zip(places, rows):
                pool[:, to[0], :, to[1]] = r
