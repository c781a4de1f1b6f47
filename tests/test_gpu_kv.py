"""The operators on the paged cache on the GPU, through the C ABI, against the oracle in float64 (oracle/qk_oracle_kv.py): rows with
several rotation axes, attention over packed prompts and drafted trees, the pages' books, a serving sequence of all of them,
captured graphs, streams, and larger sizes against a plain evaluation on the device in 64 bits."""
import numpy as np
import pytest

import kv_cases as KC

pytestmark = pytest.mark.gpu


@pytest.fixture
def up(dev):
    import torch
    return lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)


@pytest.fixture
def ws(dev):
    import torch
    return lambda n: torch.empty(n, dtype=torch.uint8, device=dev)


@pytest.mark.parametrize("case", KC.PREP, ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}x{c[3]}-p{c[4]}-r{c[5]}")
def test_prep_axes(qk, up, case):
    KC.prep_case(qk, up, case)


@pytest.mark.parametrize("case", KC.ATT, ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}x{c[3]}-p{c[4]}-b{c[9]}")
def test_attention(qk, up, ws, case):
    KC.att_case(qk, up, ws, case)


@pytest.mark.parametrize("name,case,edit,behind", KC.ODD, ids=[c[0] for c in KC.ODD])
def test_attention_odd(qk, up, ws, name, case, edit, behind):
    KC.att_case(qk, up, ws, case, edit=edit, behind=behind, l2=KC.ODD_L2.get(name, 4e-6))


@pytest.mark.parametrize("seed,page", [(0, 16), (1, 16), (2, 32), (3, 0), (5, 64)])
def test_books(qk, up, ws, seed, page):
    KC.books_case(qk, up, ws, type_=("f32", "f16")[seed % 2], dh=(128, 256)[seed // 2 % 2], page=page, seed=seed, steps=30)


def test_books_of_many_sequences(qk, up, ws):
    """More sequences and pages than the books' workgroup has threads."""
    KC.books_case(qk, up, ws, type_="f16", page=16, n_seq=1100, n_page=4000, steps=6, seed=11, layers=1, hkv=1)


@pytest.mark.parametrize("type_,dh,hq,hkv,page", [("f32", 256, 16, 2, 16), ("f16", 128, 4, 1, 0), ("f16", 256, 8, 8, 16), ("f32", 128, 10, 2, 0)])
def test_serving_sequence(qk, up, ws, dev, type_, dh, hq, hkv, page):
    import torch
    KC.serve_case(qk, up, ws, type_, dh, hq, hkv, page, sync=torch.cuda.synchronize)


def test_calls_without_work(qk, up, ws):
    KC.nothing_case(qk, up, ws)


def test_same_cache_as_the_slot_kernels(qk, dev, ws):
    """The slot kernels' caches are a slot cache of one layer: a tree of one node is qkk_attn_decode's step, a packed prompt
    qkk_attn_seq's.  1e-5 of the largest value is what the slot kernels' own forms are held to between each other."""
    import torch
    g = torch.Generator(dev).manual_seed(5)
    rnd = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    k, v = rnd(3, 2, 700, 256), rnd(3, 2, 700, 256)
    cache = qk.KvCache(k[None], v[None])
    q, qfull, at = rnd(3, 16, 256), rnd(3, 16, 512), (699, 0, 130)
    runs = qk.KvRuns(3, i32(0, 1, 2, 3), i32(0, 1, 2), i32(*at), max_run=1)
    room = [ws(b).zero_() for b in (qk.attn_runs_workspace_bytes(cache, runs, 16), qk.attn_workspace_bytes(64, 16))]
    mine = qk.attn_tree(cache, 0, runs, i32(-1, -1, -1), q, room[0], qfull=qfull)
    theirs = qk.attn_decode(q, k, v, qfull, i32(*at), room[1])
    assert (mine - theirs).abs().max() <= 1e-5 * theirs.abs().max()
    n, base = 60, 333
    q, qfull = rnd(n, 16, 256), rnd(n, 16, 512)
    runs = qk.KvRuns(n, i32(0, n), i32(2), i32(base))
    room = [ws(b).zero_() for b in (qk.attn_runs_workspace_bytes(cache, runs, 16), qk.attn_workspace_bytes(64, 16))]
    mine = qk.attn_packed(cache, 0, runs, q, room[0], qfull=qfull)
    theirs = qk.attn_decode(q, k[2:], v[2:], qfull, torch.arange(base, base + n, dtype=torch.int32, device=dev), room[1], seq=True)
    assert (mine - theirs).abs().max() <= 1e-5 * theirs.abs().max()


# ---- larger sizes, against the definition in 64 bits on the device -----------------------------------------------------

def exact(cache, layer, runs, lens, past, q, gate, parent):
    """softmax(q K / sqrt(dh)) V per run in float64, the rows gathered through the table."""
    import torch
    hq, dh = q.shape[1:]
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    lo = 0
    for s, (n, p) in enumerate(zip(lens, past)):
        total = p + n
        pages = [s] if cache.table is None else cache.table[s, :-(-total // cache.page_rows)].tolist()
        see = torch.arange(total, device=q.device) <= p + torch.arange(n, device=q.device)[:, None]
        if parent is not None:
            kin = torch.eye(n, dtype=torch.bool, device=q.device)
            up = parent[lo:lo + n].tolist()
            for i in range(n):
                if 0 <= up[i] < i:
                    kin[i] |= kin[up[i]]
            see[:, p:] = kin
        for h in range(hq):
            g = h // (hq // cache.n_kv)
            k, v = (torch.cat([x[layer, i, g] for i in pages])[:total].double() for x in (cache.k, cache.v))
            sc = (q[lo:lo + n, h].double() @ k.t()) / dh ** 0.5
            w = torch.softmax(sc.masked_fill(~see, -float("inf")), dim=-1)
            out[lo:lo + n, h] = w @ v
        lo += n
    if gate is not None:
        out *= torch.sigmoid(gate[..., dh:].double())
    return out


LARGE = [
    ("f32", 256, 16, 2, 64, 2048, (700, 1, 1500, 333), (0, 900, 300, 5), True, 0),
    ("f16", 128, 32, 8, 128, 8192, (1024, 100), (6001, 3), False, 0),
    ("f16", 256, 8, 1, 16, 1024, (513, 1000), (17, 0), False, 0),
    ("f32", 128, 5, 5, 0, 1536, (1000, 129), (511, 1200), True, 0),
    ("f32", 256, 16, 2, 0, 4352, (24, 17, 1, 64, 256), (4090, 3, 2000, 1000, 4001), True, 3),
    ("f16", 128, 32, 8, 64, 40960, (64, 7), (40001, 1234), False, 4),
    ("f16", 256, 16, 2, 256, 8192, (1,) * 16, tuple(range(500, 8500, 500))[:15] + (0,), True, 1),
    ("f32", 128, 8, 8, 128, 2048, (200, 3), (1500, 0), False, 2),
]


@pytest.mark.parametrize("case", LARGE, ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}x{c[3]}-p{c[4]}-b{c[9]}")
def test_attention_large(qk, dev, up, ws, case):
    import torch
    if dev == "cpu":
        pytest.skip("too much work for the host-side build")
    type_, dh, hq, hkv, page, cap, lens, past, gated, branch = case
    rng = np.random.default_rng(dh + hq)
    n = sum(lens)
    c = KC.make_cache(rng, type_, 2, hkv, dh, page, cap, [a + b for a, b in zip(lens, past)])
    cache = KC.device_cache(qk, up, c)
    runs = qk.KvRuns(n, up(KC.starts(lens)), up(np.arange(len(lens), dtype=np.int32)), up(np.array(past, np.int32)), max_run=max(lens))
    g = torch.Generator(dev).manual_seed(1)
    q = torch.randn((n, hq, dh), generator=g, device=dev) * 1.5
    gate = torch.randn((n, hq, 2 * dh), generator=g, device=dev) if gated else None
    parent = up(KC.parents(rng, lens, branch)) if branch else None
    space = ws(qk.attn_runs_workspace_bytes(cache, runs, hq))
    call = lambda: qk.attn_tree(cache, 1, runs, parent, q, space, qfull=gate) if branch else qk.attn_packed(cache, 1, runs, q, space, qfull=gate)  # noqa: E731
    att, again = call(), call()
    assert torch.equal(att, again)   # the same bits from call to call
    want = exact(cache, 1, runs, lens, past, q, gate, parent)
    rel = float((att.double() - want).norm() / want.norm())
    print(f"[case] {case[:6]} relative error {rel:.2e}", flush=True)
    assert rel <= 4e-6
    assert float((att.double() - want).abs().max()) <= 1e-4   # values of size 1, weights off by 1e-5 at most


def test_offsets_beyond_32_bits(qk, dev, up, ws):
    """A slot cache of more than 2^32 elements: rows of the last sequence lie behind 4 G elements (17 GB of halves)."""
    import torch
    if dev == "cpu":
        pytest.skip("too large for the host-side build")
    n_page, cap = 2, 1 << 23
    k = torch.zeros((1, n_page, 2, cap, 256), dtype=torch.float16, device=dev)   # 8.6e9 elements
    v = torch.zeros((1, n_page, 2, cap, 256), dtype=torch.float16, device=dev)
    past, n = cap - 40, 5
    g = torch.Generator(dev).manual_seed(3)
    for pool in (k, v):
        pool[0, 1, :, past - 200:past + n] = torch.randn((2, 200 + n, 256), generator=g, device=dev).half()
    k[0, 1, :, :past - 200, 0] = -60000.0   # the zero rows in front are pushed out of the softmax
    cache = qk.KvCache(k, v)
    i32 = lambda a: up(np.array(a, np.int32))  # noqa: E731
    runs = qk.KvRuns(n, i32([0, n]), i32([1]), i32([past]))
    q = torch.randn((n, 4, 256), generator=g, device=dev).abs() + 0.5
    att = qk.attn_tree(cache, 0, runs, i32([-1, 0, 1, 2, 3]), q, ws(qk.attn_runs_workspace_bytes(cache, runs, 4)))
    for h in range(4):
        kk, vv = (pool[0, 1, h // 2, past - 200:past + n].double() for pool in (k, v))
        sc = q[:, h].double() @ kk.t() / 16
        sc.masked_fill_(torch.arange(200 + n, device=dev) > 200 + torch.arange(n, device=dev)[:, None], -float("inf"))
        want = torch.softmax(sc, -1) @ vv
        assert float((att[:, h].double() - want).norm() / want.norm()) <= 4e-6
    kin = torch.randn((n, 2, 256), generator=g, device=dev)
    ones, rope = torch.ones(256, device=dev), up(qk.rope_table(4, 64))
    qk.attn_prep_axes(cache, 0, runs, q, kin, kin, ones, ones, rope, up(qk.rope_axes(64, (32,))), i32([[0] * n]))
    assert torch.equal(v[0, 1, :, past:past + n], kin.half().transpose(0, 1))
    assert torch.equal(v[0, 0], torch.zeros_like(v[0, 0]))
    qk.kv_compact(cache, i32([1]), i32([past]), i32([[2, 4]]), i32([2]))
    assert torch.equal(v[0, 1, :, past:past + 2], kin.half().transpose(0, 1)[:, [2, 4]])


# ---- streams and graphs -------------------------------------------------------------------------------------------------

def test_captured_step(qk, dev, up, ws):
    """A decode step -- grow, prepare, attend a tree, compact -- captured once, replayed while the sequences grow: every replay against
    the same calls made eagerly on a copy, with eager work between the replays."""
    import torch
    if dev == "cpu":
        pytest.skip("needs torch's graphs")
    rng = np.random.default_rng(2)
    dh, hq, hkv, page, layers = 128, 8, 2, 16, 2
    c = KC.make_cache(rng, "f16", layers, hkv, dh, page, 256, [40, 3, 100], spare=40, poison=False)
    lens, n = (4, 1, 3), 8
    parent = up(np.array([-1, 0, 0, 1, -1, -1, 0, 0], np.int32))
    ones, rope = torch.ones(dh, device=dev), up(qk.rope_table(256, 64))
    axis = up(qk.rope_axes(64, (12, 10, 10), True))
    path, n_path = up(np.array([[0, 1, 3], [0, -1, -1], [0, 2, -1]], np.int32)), up(np.array([3, 1, 2], np.int32))
    seq, start = up(np.arange(3, dtype=np.int32)), up(KC.starts(lens))
    count = up(np.array(lens, np.int32))

    class Step:
        def __init__(self):
            self.cache = KC.device_cache(qk, up, c)
            self.pos, self.want = self.cache.len.clone(), self.cache.len.clone()
            self.q, self.kin, self.vin = (torch.zeros(s, device=dev) for s in ((n, hq, 2 * dh), (n, hkv, dh), (n, hkv, dh)))
            self.axis_pos = torch.zeros((3, n), dtype=torch.int32, device=dev)
            self.runs = qk.KvRuns(n, start, seq, self.pos, max_run=4)
            self.books, self.space = ws(qk.kv_workspace_bytes(self.cache)), ws(qk.attn_runs_workspace_bytes(self.cache, self.runs, hq))
            self.att = torch.zeros((layers, n, hq, dh), device=dev)
            self.qhat = torch.zeros((n, hq, dh), device=dev)
            self.status = torch.zeros(1, dtype=torch.int32, device=dev)

        def __call__(self):
            torch.add(self.pos, count, out=self.want)
            qk.kv_resize(self.cache, self.want, self.books, status=self.status)
            for layer in range(layers):
                qk.attn_prep_axes(self.cache, layer, self.runs, self.q, self.kin, self.vin, ones, ones, rope, axis, self.axis_pos, qhat=self.qhat)
                qk.attn_tree(self.cache, layer, self.runs, parent, self.qhat, self.space, qfull=self.q, att=self.att[layer])
            qk.kv_compact(self.cache, seq, self.pos, path, n_path)
            self.pos.add_(n_path)

        def fill(self, i):
            g = torch.Generator(dev).manual_seed(i)
            for t in (self.q, self.kin, self.vin):
                t.copy_(torch.randn(t.shape, generator=g, device=dev))
            self.axis_pos.copy_(torch.randint(0, 256, (3, n), generator=g, device=dev))

    eager, held = Step(), Step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):   # warm up on a third set of buffers
        Step()()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held()
    # capturing ran nothing: both start from the same books
    for i in range(6):
        for s in (eager, held):
            s.fill(i)
        eager()
        torch.randn(1000, device=dev).sum()
        graph.replay()
        torch.cuda.synchronize()
        assert int(eager.status) == int(held.status) == 0
        assert torch.equal(eager.att, held.att), i
        for a in ("k", "v", "table", "ref", "len"):
            assert torch.equal(getattr(eager.cache, a), getattr(held.cache, a)), (i, a)


def test_side_stream(qk, dev, up, ws):
    """The calls go to torch's current stream: on a side stream, behind work that is still running there."""
    import torch
    if dev == "cpu":
        pytest.skip("needs streams")
    case = KC.ATT[4]
    rng = np.random.default_rng(0)
    type_, dh, hq, hkv, page, cap, lens, past, gated, _ = case
    c = KC.make_cache(rng, type_, 1, hkv, dh, page, cap, [a + b for a, b in zip(lens, past)])
    cache = KC.device_cache(qk, up, c)
    runs = qk.KvRuns(sum(lens), up(KC.starts(lens)), up(np.arange(3, dtype=np.int32)), up(np.array(past, np.int32)))
    q = torch.randn((sum(lens), hq, dh), device=dev)
    space = ws(qk.attn_runs_workspace_bytes(cache, runs, hq))
    want = qk.attn_packed(cache, 0, runs, q, space)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        big = torch.randn((4096, 4096), device=dev)
        late = torch.zeros_like(q)
        for _ in range(8):
            big = big @ big / 64
        late.copy_(q + 0 * big[0, 0].nan_to_num(0, 0, 0))
        got = qk.attn_packed(cache, 0, runs, late, space)
    side.synchronize()
    assert torch.equal(got, want)


# ---- the range of values -----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("name,case,edit", KC.RANGE_SCORE, ids=[c[0] for c in KC.RANGE_SCORE])
def test_scores_of_far_keys_and_queries(qk, up, ws, name, case, edit):
    KC.range_case(qk, up, ws, case, edit, "row")


@pytest.mark.parametrize("name,case,edit", KC.RANGE_SUM, ids=[c[0] for c in KC.RANGE_SUM])
def test_value_rows_of_any_size_keep_their_weight(qk, up, ws, name, case, edit):
    KC.range_case(qk, up, ws, case, edit, "row")


@pytest.mark.parametrize("name,case,edit,per", KC.RANGE_SPLIT, ids=[c[0] for c in KC.RANGE_SPLIT])
def test_small_elements_beside_large_ones(qk, up, ws, name, case, edit, per):
    KC.range_case(qk, up, ws, case, edit, per)


@pytest.mark.parametrize("case", KC.MANY_RUNS, ids=lambda c: f"{c[0]}-{len(c[6])}-b{c[9]}")
def test_attention_of_many_runs(qk, up, ws, case):
    KC.att_case(qk, up, ws, case, behind=1)


@pytest.mark.parametrize("case", KC.MANY_RUNS_PREP, ids=lambda c: f"{c[0]}-{len(c[9])}")
def test_prep_of_many_runs(qk, up, case):
    KC.prep_case(qk, up, case)
