"""Cases and checks of the operators on the paged cache, shared by the tests on the host-side kernel build (guard-paged tensors) and
those on a device.  `up` takes a numpy array to where the kernels run, `ws` makes a workspace of so many bytes.

Tolerances, with u = 2^-24 (half a step of fp32, relative):
 prep    the sum of squares of a head adds 256 values in a tree of at most 10 levels (10 u), the scale takes a division, a root and
         an addition (3 u, halved by the root), the two products 2 u, the rotation two products, an addition and the table's
         own value: each output is off by less than 16 u times the larger of its pair, which is at most sqrt(2) times the pair's
         length: 24 u = 1.4e-6 of the row's largest pair; 2e-6 of the row's maximum is asked.  In a half-precision cache
         one rounding more: 2^-11 of the value (2^-25 where halves are subnormal).
 att     a score is a sum of dh products.  Products of operands held as two halves each are exact to 2^-21 of their size, an
         fp32 sum of n of them to sqrt(n) u for the rounding of its partial sums (a random walk; 4 sigma: 4 sqrt(768) u ~ 110 u).
         With S = max over the keys of sum_d |q_d k_d| / sqrt(dh) a score is off by less than d = S * 128 u, a weight by the
         factor exp(d) - 1 ~ d, an output by 2 d * max |v|; exp, the sums over the keys and the last division
         add 64 u * max |v|.  That is the bound per element; S counts every sign against us, so in the mean the error
         is far smaller: over the whole result (2-norm) its relative size is asked to be below 4e-6 for scores of this size
         (rms of a score's error: sqrt(sum (q k)^2) / sqrt(dh) * 2^-21 < 1.5 * 4.8e-7 = 7e-7; five times that)."""
import os
import sys

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "oracle"))
import qk_oracle_kv as OK  # noqa: E402

U = 2.0 ** -24
NP = {"f32": np.float32, "f16": np.float16}


def make_cache(rng, type_, n_layer, hkv, dh, page, cap, held, spare=3, poison=True):
    """numpy pools (rows that no sequence holds are NaN when `poison`), a table of pages in random order, ref, len.
    page 0: a slot cache of cap rows per sequence."""
    n_seq, rows = len(held), page or cap
    per = cap // rows
    need = [-(-h // rows) for h in held]
    n_page = sum(need) + spare if page else n_seq
    shape = (n_layer, n_page, hkv, rows, dh)
    k, v = (rng.standard_normal(shape).astype(NP[type_]) for _ in range(2))
    table = ref = None
    if page:
        order = rng.permutation(n_page)
        table = np.full((n_seq, per), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            table[s, :n] = order[at:at + n]
            at += n
        ref = np.zeros(n_page, np.int32)
        ref[order[:at]] = 1
    if poison:
        keep = np.zeros((n_page, rows), bool)
        for s, h in enumerate(held):
            for r in range(h):
                keep[table[s, r // rows] if page else s, r % rows if page else r] = True
        for pool in (k, v):
            pool.transpose(0, 2, 1, 3, 4)[:, :, ~keep] = np.nan
    return dict(k=k, v=v, table=table, ref=ref, len=np.array(held, np.int32))


def device_cache(qk, up, c):
    opt = lambda a: None if a is None else up(a)  # noqa: E731
    return qk.KvCache(up(c["k"]), up(c["v"]), table=opt(c["table"]), ref=opt(c["ref"]), len=up(c["len"]))


def oracle_cache(c):
    lists = lambda a: None if a is None else a.tolist()  # noqa: E731
    return OK.Cache(c["k"].copy(), c["v"].copy(), lists(c["table"]), lists(c["ref"]), c["len"].tolist())


def host(t):
    return t.detach().cpu().numpy()


def same(a, b):
    return np.array_equal(np.ascontiguousarray(a).view(np.uint8), np.ascontiguousarray(b).view(np.uint8))


def starts(lens, first=0):
    return np.cumsum([first] + list(lens)).astype(np.int32)


# ---- prep ------------------------------------------------------------------------------------------------------------

PREP = [
    # type, dh, hq, hkv, page, n_rot, sections, in turn, gated, lens, past, rows behind the last run
    ("f32", 256, 16, 2, 0, 64, (11, 11, 10), False, True, (1, 1, 1), (5, 0, 31), 0),
    ("f16", 128, 8, 2, 16, 128, (24, 20, 20), True, False, (7, 0, 1, 20), (0, 3, 15, 16), 2),
    ("f32", 128, 3, 3, 32, 6, (1, 1, 1), True, True, (33,), (0,), 0),
    ("f16", 256, 5, 1, 16, 256, (128,), False, True, (2, 3), (62, 0), 1),
    ("f32", 256, 2, 1, 16, 2, (0, 1), False, False, (4,), (30,), 0),
]


def prep_case(qk, up, case, seed=0):
    type_, dh, hq, hkv, page, n_rot, sections, in_turn, gated, lens, past, behind = case
    rng = np.random.default_rng(seed + dh + hq + len(lens))
    cap, n = 64, sum(lens) + behind
    c = make_cache(rng, type_, 2, hkv, dh, page, cap, [min(a + b, cap) for a, b in zip(lens, past)], poison=False)
    ora, cache = oracle_cache(c), device_cache(qk, up, c)
    axis = qk.rope_axes(n_rot, sections, in_turn)
    assert axis.tolist() == OK.rope_axes(sections, in_turn)
    q = rng.standard_normal((n, hq, dh * (2 if gated else 1))).astype(np.float32) * 3
    kin, vin = (rng.standard_normal((n, hkv, dh)).astype(np.float32) for _ in range(2))
    qn, kn = ((1 + 0.2 * rng.standard_normal(dh)).astype(np.float32) for _ in range(2))
    rope = qk.rope_table(50, n_rot)
    axis_pos = rng.integers(-2, 60, (len(sections), n)).astype(np.int32)   # some outside the table: clamped
    st, seq, pos = starts(lens), np.arange(len(lens), dtype=np.int32), np.array(past, np.int32)
    runs = qk.KvRuns(n, up(st), up(seq), up(pos), max_run=max(lens))
    qhat = up(np.full((n, hq, dh), 7.0, np.float32))
    qk.attn_prep_axes(cache, 1, runs, up(q), up(kin), up(vin), up(qn), up(kn), up(rope), up(axis), up(axis_pos), eps=1e-6, qhat=qhat)
    want = OK.prep_axes(ora, 1, list(OK.runs(n, st, seq, pos, ora, max(lens))), q, kin, vin, qn, kn, rope, axis, axis_pos, dh, 1e-6)
    got = host(qhat)
    for r in range(n):
        if np.isnan(want[r]).all():
            assert (got[r] == 7.0).all(), r   # in no run: left as it was
        else:
            assert np.abs(got[r] - want[r]).max() <= 2e-6 * np.abs(want[r]).max(), r
    gk, gv = host(cache.k), host(cache.v)
    assert same(gv, ora.v)                     # values are copies (rounded to the cache's type), nothing else is written
    changed = ora.k != c["k"]
    assert same(np.where(changed, 0, gk), np.where(changed, 0, ora.k))
    big = np.abs(ora.k[changed].astype(np.float64)).max()
    off = np.abs(gk[changed].astype(np.float64) - ora.k[changed].astype(np.float64))
    # a half may be rounded the other way where the two lie on either side of a midpoint: one whole step
    assert (off <= 2e-6 * big + (0 if type_ == "f32" else 2.0 ** -10) * np.abs(ora.k[changed].astype(np.float64)) + 2.0 ** -24 * (type_ == "f16")).all()


# ---- attention -------------------------------------------------------------------------------------------------------

ATT = [
    # type, dh, hq, hkv, page, cap, lens, past, gated, branch (0: packed)
    ("f32", 256, 16, 2, 0, 128, (1, 1, 1), (0, 63, 127), True, 1),
    ("f16", 128, 8, 2, 16, 96, (1, 1, 1, 1), (0, 15, 16, 95), False, 1),
    ("f32", 128, 4, 4, 16, 160, (9, 1, 12), (0, 70, 130), True, 2),
    ("f16", 256, 8, 1, 32, 192, (33, 5), (100, 31), True, 3),
    ("f32", 256, 10, 2, 64, 256, (40, 0, 3), (0, 10, 250), False, 0),
    ("f16", 128, 7, 1, 16, 224, (70, 1, 17), (3, 200, 0), False, 0),
    ("f32", 128, 6, 2, 0, 176, (130, 65), (1, 64), True, 0),
    ("f16", 256, 2, 2, 128, 384, (129, 64), (200, 0), True, 0),
]


def parents(rng, lens, branch):
    return np.array([-1 if i == 0 else max(0, (i - 1) // branch - int(rng.integers(0, 2))) for n in lens for i in range(n)], np.int32)


def bound(cache, layer, rows, q, K_scale=1.0):
    """Per-element bound of the comment above, for the largest S of all rows and keys (finite ones)."""
    k = np.abs(np.nan_to_num(cache.k[layer].astype(np.float64), nan=0, posinf=0, neginf=0))
    v = np.abs(np.nan_to_num(cache.v[layer].astype(np.float64), nan=0, posinf=0, neginf=0))
    s = max(float((np.abs(q[r].astype(np.float64)).max(0) * k.max((0, 1, 2))).sum()) for r in {r for r, *_ in rows}) / np.sqrt(q.shape[2])
    return (2 * 128 * U * s + 64 * U) * v.max()


def check_att(got, want, tol, rows, untouched=7.0, l2=4e-6):
    live = np.zeros(got.shape[0], bool)
    live[[r for r, *_ in rows]] = True
    assert (got[~live] == untouched).all()
    fin = np.isfinite(want[live])
    assert np.isfinite(got[live][fin]).all()
    off = np.abs(got[live][fin] - want[live][fin])
    assert off.max() <= tol, (off.max(), tol)
    rel = np.linalg.norm(off) / max(np.linalg.norm(want[live][fin]), 1e-30)
    assert rel <= l2, rel
    assert not np.isfinite(got[live][~fin]).any()


def att_case(qk, up, ws, case, seed=0, poison=True, edit=None, behind=0, l2=4e-6, q_scale=1.5, wide=None):
    """One call on a cache whose unheld rows are NaN, against the oracle.  edit(dict): changes the inputs first."""
    type_, dh, hq, hkv, page, cap, lens, past, gated, branch = case
    rng = np.random.default_rng(seed + dh + hq + sum(lens))
    n = sum(lens) + behind
    c = make_cache(rng, type_, 2, hkv, dh, page, cap, [min(a + b, cap) for a, b in zip(lens, past)], poison=poison)
    x = dict(c=c, start=starts(lens), seq=np.arange(len(lens), dtype=np.int32), pos=np.array(past, np.int32),
             q=(rng.standard_normal((n, hq, dh)) * q_scale).astype(np.float32), gate=rng.standard_normal((n, hq, 2 * dh)).astype(np.float32) if gated else None,
             parent=np.concatenate([parents(rng, lens, branch), np.full(behind, -1, np.int32)]) if branch else None, max_run=max(lens))
    if edit:
        edit(x)
    cache, ora = device_cache(qk, up, c), oracle_cache(c)
    runs = qk.KvRuns(n, up(x["start"]), up(x["seq"]), up(x["pos"]), max_run=x["max_run"])
    att = up(np.full((n, hq, dh), 7.0, np.float32))
    space = ws(qk.attn_runs_workspace_bytes(cache, runs, hq))
    qf = None if x["gate"] is None else up(x["gate"])
    if branch:
        qk.attn_tree(cache, 1, runs, up(x["parent"]), up(x["q"]), space, qfull=qf, att=att)
    else:
        qk.attn_packed(cache, 1, runs, up(x["q"]), space, qfull=qf, att=att)
    rows = list(OK.runs(n, x["start"], x["seq"], x["pos"], ora, x["max_run"]))
    with np.errstate(all="ignore"):
        want = OK.attend(ora, 1, rows, x["q"], x["gate"], x["parent"])
    got = host(att)
    if rows:
        check_att(got, want, bound(ora, 1, rows, x["q"]), rows, l2=l2)
    else:
        assert (got == 7.0).all()
    assert same(host(cache.k), c["k"]) and same(host(cache.v), c["v"])
    return got, want


def place(c, seq, r):
    page = c["k"].shape[3]
    return (seq, r) if c["table"] is None else (int(c["table"][seq, r // page]), r % page)


# ---- books -----------------------------------------------------------------------------------------------------------

def check_books(cache, ora):
    assert same(host(cache.len), np.array(ora.length, np.int32))
    if ora.table is not None:
        assert same(host(cache.table), np.array(ora.table, np.int32)) and same(host(cache.ref), np.array(ora.ref, np.int32))
    assert same(host(cache.k), ora.k) and same(host(cache.v), ora.v)


def check_invariant(ora):
    """Every page is held as often as its count says, and a sequence's pages are those of its length."""
    held = np.zeros(ora.n_page, int)
    for row, n in zip(ora.table, ora.length):
        pages = [p for p in row if p >= 0]
        assert len(pages) == -(-n // ora.page_rows)
        for p in pages:
            held[p] += 1
    assert held.tolist() == ora.ref


def books_case(qk, up, ws, type_="f32", dh=128, page=16, n_seq=6, n_page=14, steps=12, seed=0, layers=2, hkv=2):
    """A random walk of resizes, forks and compactions, books and rows compared after every call."""
    rng = np.random.default_rng(seed)
    per = 5
    c = make_cache(rng, type_, layers, hkv, dh, page, per * (page or 16), [0] * n_seq, spare=n_page, poison=False)
    cache, ora = device_cache(qk, up, c), oracle_cache(c)
    space = ws(qk.kv_workspace_bytes(cache))
    seen = set()
    for step in range(steps):
        what = rng.integers(0, 3) if step else 0
        if what == 0:
            new = [int(rng.choice([-1, 0, rng.integers(0, ora.cap + 1), min(n + 1, ora.cap)])) for n in ora.length]
            if step == steps - 2:
                new[-1] = ora.cap + 1
            if step == steps - 1:
                new = [ora.cap] * n_seq
            got, want = qk.kv_resize(cache, up(np.array(new, np.int32)), space), OK.resize(ora, new)
            seen.add(("resize", int(np.sign(want))))
        elif what == 1:
            empty = [s for s, n in enumerate(ora.length) if n == 0]
            n = int(rng.integers(0, len(empty) + 1))
            dst, src = empty[:n], [int(s) for s in rng.integers(0, n_seq, n)]
            if rng.random() < 0.15:
                src, dst = src + [0], dst + [int(rng.integers(-1, n_seq + 1))]
                if len(dst) > n_seq:
                    src, dst = src[:n_seq], dst[:n_seq]
            i32 = lambda a: up(np.array(a, np.int32))  # noqa: E731
            got, want = qk.kv_fork(cache, i32(src), i32(dst), space), OK.fork(ora, src, dst)
            seen.add(("fork", want))
        else:
            seqs = [s for s, n in enumerate(ora.length) if n > 1 and (ora.table is None or all(ora.ref[p] == 1 for p in ora.table[s] if p >= 0))]
            base = [int(rng.integers(0, ora.length[s])) for s in seqs]
            wide = 7
            path, count = np.full((len(seqs), wide), -1, np.int32), []
            for i, (s, b) in enumerate(zip(seqs, base)):
                m = min(ora.length[s] - b, wide, 1 + int(rng.integers(0, wide)))
                path[i, :m] = np.sort(rng.choice(ora.length[s] - b, m, replace=False))
                count.append(m)
            if len(seqs) > 1:   # one that is not ascending: left out
                path[0, :2], count[0] = (1, 1), 2
            if seqs:
                qk.kv_compact(cache, *(up(np.array(a, np.int32)) for a in (seqs, base)), up(path), up(np.array(count, np.int32)))
                OK.compact(ora, seqs, base, path.tolist(), count)
            got = want = None
        if got is not None:
            assert int(host(got)[0]) == want, (step, what)
        check_books(cache, ora)
        if ora.table is not None:
            check_invariant(ora)
    return seen


# ---- a serving sequence ------------------------------------------------------------------------------------------------

def serve_case(qk, up, ws, type_, dh, hq, hkv, page, prompt=21, sync=lambda: None):
    """Two prompts packed into one pass, one forked twice, trees drafted on all four sequences, a path accepted, the next token: every
    attention result and the whole cache against the oracle, which keeps a cache of its own."""
    rng = np.random.default_rng(dh + hq + page)
    layers, n_seq, cap, n_rot = 2, 4, 64, 32
    c = make_cache(rng, type_, layers, hkv, dh, page, cap, [0] * n_seq, spare=14, poison=False)
    cache, ora = device_cache(qk, up, c), oracle_cache(c)
    book_ws = ws(qk.kv_workspace_bytes(cache))
    i32 = lambda a: up(np.array(a, np.int32))  # noqa: E731
    axis, rope = qk.rope_axes(n_rot, (6, 5, 5), True), qk.rope_table(cap, n_rot)
    qn, kn = ((1 + 0.2 * rng.standard_normal(dh)).astype(np.float32) for _ in range(2))
    axis_d, rope_d, qn_d, kn_d = up(axis), up(rope), up(qn), up(kn)

    def pass_(seqs, lens, past, parent=None):
        n, st = sum(lens), starts(lens)
        runs = qk.KvRuns(n, up(st), i32(seqs), i32(past), max_run=max(lens))
        space = ws(qk.attn_runs_workspace_bytes(cache, runs, hq))
        rows = list(OK.runs(n, st, seqs, past, ora, max(lens)))
        for layer in range(layers):
            q = rng.standard_normal((n, hq, 2 * dh)).astype(np.float32)
            kin, vin = (rng.standard_normal((n, hkv, dh)).astype(np.float32) for _ in range(2))
            t = np.array([p + i for m, p in zip(lens, past) for i in range(m)])
            axis_pos = np.stack([t, t // 3, t % 7]).astype(np.int32)
            qd = up(q)
            qhat = qk.attn_prep_axes(cache, layer, runs, qd, up(kin), up(vin), qn_d, kn_d, rope_d, axis_d, up(axis_pos))
            if parent is None:
                att = qk.attn_packed(cache, layer, runs, qhat, space, qfull=qd)
            else:
                att = qk.attn_tree(cache, layer, runs, i32(parent), qhat, space, qfull=qd)
            sync()
            OK.prep_axes(ora, layer, rows, q, kin, vin, qn, kn, rope, axis, axis_pos, dh, 1e-6)
            # the rows the kernels wrote are what the next attention reads, in the oracle too (a half may differ by a step)
            gk = host(cache.k).astype(np.float64)
            assert np.nanmax(np.abs(gk - ora.k.astype(np.float64))) <= (2e-5 if type_ == "f32" else 2.0 ** -8)
            ora.k[...] = host(cache.k)
            want = OK.attend(ora, layer, rows, host(qhat), q, parent)
            check_att(host(att), want, bound(ora, layer, rows, host(qhat)), rows)

    def books(f, *a):
        got, want = getattr(qk, "kv_" + f)(cache, *[i32(x) for x in a], book_ws), getattr(OK, f)(ora, *[list(x) for x in a])
        assert int(host(got)[0]) == want == 0, f
        check_books(cache, ora)

    books("resize", [prompt, 0, 9, 0])
    pass_([0, 2], [prompt, 9], [0, 0])
    books("fork", [0, 0], [1, 3])
    held = [prompt, prompt, 9, prompt]
    books("resize", [h + 5 for h in held])              # the three that share a part-filled page each get a copy
    tree = [-1, 0, 0, 1, 2]
    pass_([0, 1, 2, 3], [5] * 4, held, tree * 4)
    path, count = [[0, 1, 3], [0, 2, 4], [0, 2, -1], [0, -1, -1]], [3, 3, 2, 1]
    qk.kv_compact(cache, i32([0, 1, 2, 3]), i32(held), i32(path), i32(count))
    OK.compact(ora, [0, 1, 2, 3], held, path, count)
    check_books(cache, ora)
    books("resize", [h + n + 1 for h, n in zip(held, count)])   # rejected rows cut off, room for the next token
    pass_([3, 1, 0, 2], [1] * 4, [held[s] + count[s] for s in (3, 1, 0, 2)], [-1] * 4)
    books("resize", [0, -1, 0, -1])
    books("resize", [0] * 4)
    if page:
        assert not any(ora.ref)


# ---- calls at the edges: what a row does not see, runs out of range, rows in no run -------------------------------------

def _poison_later(x):
    """The last row of the first run holds infinities and NaN: no earlier row may show them, the last row must."""
    c = x["c"]
    n, p = int(x["start"][1]), int(x["pos"][0])
    page, r = place(c, 0, p + n - 1)
    c["v"][1, page, :, r, ::3] = np.inf
    c["v"][1, page, :, r, 1::3] = np.nan
    c["k"][1, page, :, r, 5] = np.nan


def _poison_cousin(x):
    """A node that is nobody's ancestor holds NaN: only its own row may show it."""
    c, n, p = x["c"], int(x["start"][1]), int(x["pos"][0])
    x["parent"][:n] = [-1] + [0] * (n - 1)
    page, r = place(c, 0, p + 1)
    c["v"][1, page, :, r] = np.nan
    c["k"][1, page, :, r] = -np.inf


def _no_pages(x):
    """No page at all for the first sequence (its rows see nothing: zeros), one missing page in the middle of the second's."""
    x["c"]["table"][0] = -1
    x["c"]["table"][1, 1] = 1 << 20


def _bad_runs(x):
    """Sequences and positions out of range: their rows are left as they were."""
    x["seq"][0], x["pos"][1] = 77, -4
    x["seq"][2], x["pos"][3] = -1, 1 << 30


def _cut(x):
    """Runs longer than max_run are cut there; the last row of the batch lies in no run."""
    x["max_run"] = 4
    x["start"][-1] -= 1


def _past_the_end(x):
    """Rows behind the sequence's last page see what there is."""
    x["pos"][0] = 94


def _same_sequence(x):
    """Two runs of one sequence at different positions (a prompt cut into two runs of one pass)."""
    x["seq"][:], x["pos"][:] = 1, (0, 20)


def _bad_parents(x):
    """Parents that point at the node itself, ahead, or far outside: roots."""
    x["parent"][1], x["parent"][2], x["parent"][3], x["parent"][4] = 1, 4, 1 << 30, -9


def _large(x):
    """Values far outside a half's range, and keys of very different size from row to row."""
    c = x["c"]
    c["v"] *= np.float32(3e6)
    c["k"] *= (10.0 ** np.linspace(-6, 0, c["k"].shape[3])).astype(np.float32)[None, None, None, :, None]


def _small(x):
    """Values far below a half's smallest."""
    x["c"]["v"] *= np.float32(1e-12)
    x["c"]["k"] *= np.float32(1e3)
    x["q"] *= np.float32(1e-3)


def _mixed_values(x):
    """Neighbouring rows whose values differ by ten orders of magnitude."""
    c = x["c"]
    c["v"] *= (10.0 ** (np.arange(c["v"].shape[3]) % 3 * 5.0 - 5)).astype(np.float32)[None, None, None, :, None]


def _peaked(x):
    """Scores of several hundred: the running maximum has to follow."""
    x["q"] *= np.float32(40)


def _zero_values(x):
    """Rows of zeros among the keys and values, and a query of zeros."""
    x["c"]["v"][:, :, :, 3::4] = 0
    x["c"]["k"][:, :, :, ::5] = 0
    x["q"][0] = 0


ODD = [
    ("later rows not finite, packed", ("f32", 256, 4, 2, 16, 96, (20, 3), (30, 5), True, 0), _poison_later, 0),
    ("later rows not finite, packed, half", ("f16", 128, 3, 1, 16, 96, (37, 3), (0, 5), False, 0), _poison_later, 1),
    ("later rows not finite, packed, many rows", ("f32", 128, 8, 1, 16, 96, (40, 3), (30, 5), False, 0), _poison_later, 0),
    ("cousin not finite", ("f32", 256, 4, 2, 0, 64, (5, 2), (30, 5), False, 2), _poison_cousin, 0),
    ("cousin not finite, half", ("f16", 128, 8, 1, 16, 64, (5, 2), (15, 0), True, 2), _poison_cousin, 0),
    ("cousin not finite, wide", ("f16", 256, 8, 1, 16, 96, (40, 2), (15, 0), True, 2), _poison_cousin, 0),
    ("sequences without pages", ("f32", 128, 4, 2, 16, 96, (3, 2, 4), (20, 40, 1), True, 1), _no_pages, 0),
    ("sequences without pages, packed", ("f16", 256, 4, 4, 16, 96, (3, 40, 4), (20, 40, 1), False, 0), _no_pages, 0),
    ("runs out of range", ("f32", 128, 4, 2, 16, 96, (3, 2, 4, 1, 2), (20, 40, 1, 3, 4), False, 0), _bad_runs, 2),
    ("runs cut", ("f16", 128, 4, 2, 16, 96, (3, 9, 5), (20, 40, 1), True, 0), _cut, 3),
    ("past the end", ("f32", 128, 4, 2, 16, 96, (6, 2), (10, 3), False, 0), _past_the_end, 0),
    ("past the end, tree", ("f16", 128, 4, 2, 16, 96, (6, 2), (10, 3), False, 2), _past_the_end, 0),
    ("one sequence twice", ("f32", 256, 4, 2, 16, 96, (20, 10), (0, 70), False, 0), _same_sequence, 0),
    ("parents out of range", ("f32", 128, 4, 2, 16, 96, (7, 2), (20, 40), False, 2), _bad_parents, 0),
    ("values beyond half range", ("f32", 256, 4, 2, 16, 96, (20, 9), (30, 5), False, 0), _large, 0),
    ("values beyond half range, tree", ("f32", 128, 4, 2, 16, 96, (5, 9), (30, 5), False, 2), _large, 0),
    ("values below half range", ("f32", 128, 16, 2, 0, 96, (20, 9), (30, 5), False, 0), _small, 0),
    ("values below half range, tree", ("f32", 256, 4, 2, 0, 96, (1, 9), (30, 5), False, 2), _small, 0),
    ("values of very different size", ("f32", 128, 4, 1, 16, 96, (20, 9), (60, 5), False, 0), _mixed_values, 0),
    ("values of very different size, tree", ("f32", 256, 4, 1, 16, 96, (5, 9), (60, 5), False, 2), _mixed_values, 0),
    ("peaked", ("f32", 256, 4, 2, 16, 96, (20, 9), (60, 5), False, 0), _peaked, 0),
    ("peaked, half", ("f16", 128, 4, 2, 16, 96, (5, 9), (60, 5), True, 2), _peaked, 0),
    ("zeros", ("f32", 128, 4, 2, 16, 96, (20, 9), (60, 5), False, 0), _zero_values, 0),
    ("zeros, tree", ("f32", 256, 4, 2, 16, 96, (5, 9), (60, 5), False, 2), _zero_values, 0),
]
# scores forty times as large: a score's error, and with it a weight's, grows with them
ODD_L2 = {"peaked": 40 * 4e-6, "peaked, half": 40 * 4e-6}


def nothing_case(qk, up, ws):
    """Calls without rows, runs, forks or paths do nothing, though their empty tensors have no address."""
    rng = np.random.default_rng(3)
    c = make_cache(rng, "f32", 1, 2, 128, 16, 64, (20, 0))
    cache = device_cache(qk, up, c)
    i32 = lambda *s: up(np.zeros(s, np.int32))  # noqa: E731
    f32 = lambda *s: up(np.zeros(s, np.float32))  # noqa: E731
    room = ws(max(qk.kv_workspace_bytes(cache), 4096))
    for n_rows, n_run in ((0, 0), (0, 1), (3, 0)):
        runs = qk.KvRuns(n_rows, i32(n_run + 1), i32(n_run), i32(n_run))
        q, kv = f32(n_rows, 4, 128), f32(n_rows, 2, 128)
        qhat, att = up(np.full((n_rows, 4, 128), 7, np.float32)), up(np.full((n_rows, 4, 128), 7, np.float32))
        qk.attn_prep_axes(cache, 0, runs, q, kv, kv, f32(128), f32(128), f32(64, 32, 2), up(np.zeros(32, np.uint8)), i32(1, n_rows), qhat=qhat)
        qk.attn_packed(cache, 0, runs, q, room, att=att)
        qk.attn_tree(cache, 0, runs, i32(n_rows), q, room, att=att)
        assert (host(qhat) == 7).all() and (host(att) == 7).all()
    assert host(qk.kv_fork(cache, i32(0), i32(0), room)).tolist() == [0]
    qk.kv_compact(cache, i32(0), i32(0), i32(0, 4), i32(0))
    qk.kv_compact(cache, i32(1), i32(1), i32(1, 0), i32(1))
    assert same(host(cache.k), c["k"]) and same(host(cache.v), c["v"])
    assert same(host(cache.table), c["table"]) and same(host(cache.ref), c["ref"]) and same(host(cache.len), c["len"])


# ---- the range of values -----------------------------------------------------------------------------------------------

def check_range(got, want, rows, per, tol=4e-6):
    """Relative error (2-norm) of every row's heads ("row") or of every dim over all rows ("dim"): what one large row, or one large dim,
    would hide in the whole result.  The tolerance is that of the whole result at the head of this file, a bound of each element's
    own rounding errors taken for signs at random: a row's 128 or 256 elements and a dim's rows and heads are as many."""
    live = sorted({r for r, *_ in rows})
    a, b = got[live].astype(np.float64), want[live]
    assert np.isfinite(a).all()
    axis = 2 if per == "row" else (0, 1)
    off, size = np.sqrt(((a - b) ** 2).sum(axis)), np.sqrt((b ** 2).sum(axis))
    worst = (off / np.where(size > 0, size, 1)).max()
    assert worst <= tol, (per, worst)


def range_case(qk, up, ws, case, edit, per, seed=0, tol=4e-6):
    """One call whose values, keys or queries `edit` spreads over fp32's range, held to every row's or dim's own size."""
    box = {}

    def both(x):
        edit(x)
        box.update(x)
    got, want = att_case(qk, up, ws, case, seed=seed, poison=False, edit=both, l2=np.inf)
    rows = list(OK.runs(got.shape[0], box["start"], box["seq"], box["pos"], oracle_cache(box["c"]), box["max_run"]))
    check_range(got, want, rows, per, tol)


# many rows (several ranges of keys, one range, a tree) and few rows
FORMS = [("many rows", ("f32", 256, 4, 2, 16, 160, (20, 9), (90, 65), False, 0)), ("many rows, one range", ("f32", 128, 8, 1, 0, 64, (20, 9), (43, 40), True, 0)),
         ("wide tree", ("f32", 128, 8, 2, 16, 192, (20, 9), (120, 65), False, 2)), ("few rows", ("f32", 256, 4, 2, 16, 160, (5, 1), (140, 65), False, 2))]


def _far_and_apart(p):
    """Keys and queries of size 2^p that share no dim: every score is zero though the product of their sizes passes fp32's range."""
    def edit(x):
        half = x["q"].shape[2] // 2
        x["c"]["k"] *= np.float32(2.0 ** p)
        x["c"]["k"][..., :half] = 0
        x["q"] *= np.float32(2.0 ** p)
        x["q"][..., half:] = 0
    return edit


def _sizes_cancel(p):
    """Keys of size 2^p, queries of size 2^-p: ordinary scores."""
    def edit(x):
        x["c"]["k"] *= np.float32(2.0 ** p)
        x["q"] *= np.float32(2.0 ** -p)
    return edit


RANGE_SCORE = [(f"{what}, {where}", case, edit) for what, edit in [("keys and queries of size 2^70 in dims of their own", _far_and_apart(70)),
                                                                  ("keys 2^100, queries 2^-100", _sizes_cancel(100)), ("keys 2^-100, queries 2^100", _sizes_cancel(-100))]
               for where, case in FORMS]


def _rows_of_size(every, small, large):
    """Cache rows 0, every, 2 every ... have values of size `small`, the others of size `large` (as powers of two; None: zeros)."""
    def edit(x):
        for s in range(len(x["seq"])):
            for r in range(x["c"]["len"][s]):
                p = small if r % every == 0 else large
                page, at = place(x["c"], s, r)
                x["c"]["v"][:, page, :, at] *= np.float32(0 if p is None else 2.0 ** p)
    return edit


def _first_rows_zero(n, p):
    """The first n rows of a sequence are zeros, the others of size 2^p: a whole tile, or a whole range of keys, of either."""
    def edit(x):
        for s in range(len(x["seq"])):
            for r in range(x["c"]["len"][s]):
                page, at = place(x["c"], s, r)
                x["c"]["v"][:, page, :, at] *= np.float32(2.0 ** p if r >= n else 0)
    return edit


RANGE_SUM = [(f"{what}, {where}", case, edit)
             for what, edit in [("every other row zero beside 2^60", _rows_of_size(2, None, 60)), ("every other row zero beside 2^110", _rows_of_size(2, None, 110)),
                                ("every third row 2^-100 beside 2^100", _rows_of_size(3, -100, 100)), ("one row in seven 2^100 beside 2^-100", _rows_of_size(7, 100, -100)),
                                ("the first 32 rows zero, then 2^50", _first_rows_zero(32, 50)), ("the first 64 rows zero, then 2^44", _first_rows_zero(64, 44)),
                                ("the first 64 rows zero, then 2^110", _first_rows_zero(64, 110))]
             for where, case in FORMS if "64" not in what or "one range" not in where]


FORMS16 = [("halves, many rows", ("f16", 128, 8, 2, 16, 160, (20, 9), (90, 65), False, 0)), ("halves, many rows, one range", ("f16", 256, 8, 1, 0, 64, (20, 9), (43, 40), True, 0)),
           ("halves, wide tree", ("f16", 256, 8, 2, 16, 192, (20, 9), (120, 65), False, 2)), ("halves, few rows", ("f16", 128, 4, 2, 16, 160, (5, 1), (140, 65), False, 2))]


def _value_dim(p):
    """One dim of all value rows is 2^p times as large as the others."""
    def edit(x):
        x["c"]["v"][..., 0] *= np.float32(2.0 ** p)
    return edit


def _value_dim_of_a_row(p):
    """One dim of one value row is 2^p times as large as everything else."""
    def edit(x):
        for s in range(len(x["seq"])):
            page, at = place(x["c"], s, 2)
            x["c"]["v"][:, page, :, at, 5] *= np.float32(2.0 ** p)
    return edit


def _key_dim(p):
    """One dim of the keys is 2^p times as large as the others, that of the queries as much smaller."""
    def edit(x):
        x["c"]["k"][..., 0] *= np.float32(2.0 ** p)
        x["q"][..., 0] *= np.float32(2.0 ** -p)
    return edit


def _query_dim(p):
    """One dim of the queries is 2^p times as large as the others, that of the keys as much smaller."""
    def edit(x):
        x["q"][..., 0] *= np.float32(2.0 ** p)
        x["c"]["k"][..., 0] *= x["c"]["k"].dtype.type(2.0 ** -p)
    return edit


def _sink(bits):
    """The first key takes nearly the whole weight, 2^bits times that of any other, and its values are zeros."""
    def edit(x):
        c, dh = x["c"], x["q"].shape[2]
        x["q"] *= np.float32(0.05)
        x["q"][..., 1] = 8
        c["k"][..., 1] = 0
        for s in range(len(x["seq"])):
            page, at = place(c, s, 0)
            c["k"][:, page, :, at] = 0
            c["k"][:, page, :, at, 1] = bits * np.log(2) * np.sqrt(dh) / 8
            c["v"][:, page, :, at] = 0
    return edit


# Operands held as two halves are exact to 2^-22 down to 2^-16 of their row's largest and to 2^-39 of that below; a product's weights
# likewise, to 2^-36 of the row's largest.  At 2^-20 (values) and 2^-17 (weights) of the largest that is 2^-19 of the element, half of
# the 4e-6 of the whole result.
RANGE_SPLIT = [(f"{what}, {where}", case, edit, per) for what, edit, per in
               [("a value dim 2^6", _value_dim(6), "dim"), ("a value dim 2^14", _value_dim(14), "dim"), ("a value dim 2^20", _value_dim(20), "dim"),
                ("a value 2^14", _value_dim_of_a_row(14), "dim"), ("a value 2^17", _value_dim_of_a_row(17), "dim"),
                ("a key dim 2^10", _key_dim(10), "row"), ("a key dim 2^16", _key_dim(16), "row")] for where, case in FORMS]
RANGE_SPLIT += [(f"{what}, {where}", case, edit, "row") for what, edit in [("a query dim 2^10", _query_dim(10)), ("a query dim 2^14", _query_dim(14)),
                                                                           ("a key with the weight, 2^17", _sink(17))] for where, case in FORMS + FORMS16]


# ---- more runs than a wave looks over at once ------------------------------------------------------------------------------

def many_runs(n_run, seed, longest, cap):
    """Lengths and pasts of n_run runs, a third of them empty, the last ones too."""
    rng = np.random.default_rng(seed)
    lens = [int(n) if rng.random() > 0.33 else 0 for n in rng.integers(1, longest + 1, n_run)]
    lens[-2:] = [0, 0]
    lens[n_run // 2], lens[64 if n_run > 66 else 0] = longest, longest
    return tuple(lens), tuple(int(p) for p in rng.integers(0, cap - longest, n_run))


MANY_RUNS = [("f16", 128, 2, 1, 16, 160, *many_runs(65, 1, 4, 160), False, 1), ("f32", 128, 2, 1, 16, 160, *many_runs(130, 2, 3, 160), True, 2),
             ("f16", 128, 4, 1, 16, 160, *many_runs(140, 3, 11, 160), False, 0), ("f32", 128, 4, 1, 0, 160, *many_runs(100, 4, 10, 160), False, 2),
             ("f32", 128, 12, 1, 0, 48, *many_runs(70, 5, 12, 48), True, 0)]
MANY_RUNS_PREP = [("f16", 128, 2, 1, 16, 64, (11, 11, 10), True, False, many_runs(140, 6, 3, 64)[0], many_runs(140, 6, 3, 60)[1], 2),
                  ("f32", 256, 2, 1, 0, 64, (32,), False, True, many_runs(67, 7, 4, 64)[0], many_runs(67, 7, 4, 60)[1], 0)]
