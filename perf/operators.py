"""What the paged-cache operators are measured on: preparing rows with several rotation axes, attention over
packed prompts, attention of drafted token trees, and forking / compacting the cache they all share.

A case names one operator and its sizes.  `prepare` makes what a serving program has in hand, `run` makes one pass: in
elementary torch operations in 32 bits, or -- where `own` is set -- through the library's entry points.  A cache holds
keys and values [layer][page][kv head][row][dh]; sequence s finds its row r in page table[s][r / page_rows].  Without a
table (page_rows = the capacity of a slot) sequence s is page s."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16}
EPS = 1e-6


# ---- cases -------------------------------------------------------------------------------------------------------

def listed():
    return [
        # the next token of sixteen slots of the engine's attention layer (text: all three axes alike), cache per slot
        dict(name="prep_step", op="prep", type="f32", hq=16, hkv=2, dh=256, n_rot=64, sections="11,11,10", mixed=False,
             gated=True, page=0, cap=4096, lens="1," * 15 + "1", past="17,4095,300,1023,64,2047,511,1,0,900,3000,128,77,2500,640,33"),
        # prompts with images in them, packed into one pass, axes dealt out pair by pair, half-precision pages
        dict(name="prep_images", op="prep", type="f16", hq=32, hkv=8, dh=128, n_rot=128, sections="24,20,20", mixed=True,
             gated=False, page=64, cap=4096, lens="2048,1531,33,700", past="0,64,1000,7"),
        # eight short chat prompts that arrive together
        dict(name="packed_short", op="packed", type="f32", hq=16, hkv=2, dh=256, gated=True, page=64, cap=512,
             lens="37,5,128,1,300,64,17,211", past="0,0,0,0,0,0,0,0"),
        # chunks of three prompts, two of them with a long part already in the cache
        dict(name="packed_chunks", op="packed", type="f16", hq=32, hkv=8, dh=128, gated=False, page=128, cap=8192,
             lens="1024,777,2048", past="6000,0,3001"),
        # two whole long prompts of the engine's attention layer
        dict(name="packed_long", op="packed", type="f32", hq=16, hkv=2, dh=256, gated=True, page=0, cap=8192,
             lens="8191,3001", past="0,0"),
        # plain sampling: one token for each of sixteen sequences (a tree of one node)
        dict(name="tree_one", op="tree", type="f16", hq=32, hkv=8, dh=128, gated=False, page=64, cap=4096, lens="1," * 15 + "1",
             past="17,4095,300,1023,64,2047,511,1,0,900,3000,128,77,2500,640,33", branch=1),
        # one chat with a small tree behind a thousand positions
        dict(name="tree_small", op="tree", type="f32", hq=16, hkv=2, dh=256, gated=True, page=0, cap=4096, lens="8", past="1000", branch=2),
        # sixteen slots, each with a tree, at the server's context
        dict(name="tree_slots", op="tree", type="f32", hq=16, hkv=2, dh=256, gated=True, page=64, cap=4224, lens="24," * 15 + "17",
             past="4096,4000,3500,4095,2048,4001,3999,4096,1025,3333,4096,2900,4090,3700,4096,4011", branch=3),
        # two long documents with wide trees
        dict(name="tree_long", op="tree", type="f16", hq=32, hkv=8, dh=128, gated=False, page=128, cap=65536, lens="64,33",
             past="32768,65001", branch=4),
        # four prompts, each continued in four ways: children share the prompt's pages and copy the part-filled last one
        dict(name="fork_pages", op="fork", type="f16", layers=10, hkv=2, dh=256, page=64, cap=2048, lens="1000,64,333,2001", ways=3, grow=17),
        # a long prompt copied from one slot of a slot cache to others (a prefix shared by several chats)
        dict(name="fork_slots", op="fork", type="f32", layers=10, hkv=2, dh=256, page=0, cap=4096, lens="4001,1777", ways=3, grow=9),
        # the accepted path of sixteen drafted trees moved to the front, all layers
        dict(name="compact_trees", op="compact", type="f32", layers=10, hkv=2, dh=256, page=64, cap=512,
             lens="24," * 15 + "17", past="17,409,300,102,64,204,400,1,0,90,300,128,77,250,64,33", accept=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def _heads(rng):
    dh = rng.choice((128, 256))
    hkv = rng.choice((1, 2, 4, 8))
    group = rng.choice([g for g in (1, 2, 4, 5, 8) if g * hkv * dh <= 4096])
    return dict(dh=dh, hkv=hkv, hq=hkv * group, type=rng.choice(("f32", "f16")), page=rng.choice((0, 16, 64, 128, 256)))


def _text(values):
    return ",".join(str(v) for v in values)


def draw(rng):
    op = rng.choice(("prep", "packed", "tree", "fork", "compact"))
    c = dict(op=op, **_heads(rng))
    if op == "prep":
        c["n_rot"] = rng.choice((32, 64, c["dh"]))
        a, b = rng.randint(1, c["n_rot"] // 4), rng.randint(1, c["n_rot"] // 8)
        c.update(sections=_text((c["n_rot"] // 2 - a - b, a, b)), mixed=rng.random() < 0.5, gated=rng.random() < 0.5)
        n = rng.randint(1, 16)
        lens = [_log(rng, 1, 3400 // n) for _ in range(n)]
        past = [rng.choice((0, _log(rng, 1, 2000))) for _ in lens]
    elif op == "packed":
        n = rng.randint(1, 8)
        lens = [_log(rng, 1, 4096 // n) for _ in range(n)]
        past = [rng.choice((0, 0, _log(rng, 1, 4000))) for _ in lens]
        c["gated"] = rng.random() < 0.5
    elif op == "tree":
        n = rng.choice((1, 2, 3, 8, 16))
        lens = [_log(rng, 1, 64) for _ in range(n)]
        c["hkv"], c["hq"] = (1, c["hq"] // c["hkv"]) if c["hkv"] * c["dh"] > 1024 else (c["hkv"], c["hq"])
        past = [_log(rng, 1, 48000 // n) for _ in lens]
        c.update(gated=rng.random() < 0.5, branch=rng.randint(1, 5))
    else:
        c.pop("hq")
        c["hkv"] = min(c["hkv"], 4)
        c["layers"] = rng.choice([n for n in (1, 3, 10) if n * c["hkv"] * c["dh"] <= 5120])
        if op == "fork":
            n = rng.randint(1, 4)
            lens = [_log(rng, 1, 2000) for _ in range(n)]
            past = lens
            c.update(ways=rng.randint(1, 3), grow=rng.randint(1, 40))
        else:
            n = rng.randint(1, 16)
            c["accept"] = rng.randint(1, 8)
            lens = [rng.randint(1, 64) for _ in range(n)]
            past = [_log(rng, 1, 400) for _ in lens]
    if op == "fork":
        top = max(lens) + c["grow"]
        c["lens"] = _text(lens)
    else:
        top = max(a + b for a, b in zip(lens, past))
        c.update(lens=_text(lens), past=_text(past))
    c["cap"] = -(-top // 256) * 256
    return c


def _ints(text):
    return [int(v) for v in text.split(",")]


# ---- inputs ------------------------------------------------------------------------------------------------------

def _cache(case, g, n_layer, n_seq, held):
    """Pools of random rows and the table of n_seq sequences, sequence s holding held[s] rows in pages that lie in any order."""
    page = case["page"] or case["cap"]
    per = case["cap"] // page
    want = [-(-h // page) for h in held]
    if case["page"]:
        n_page = sum(want) + n_seq + 8  # some to spare: the pages that growing sequences take
    else:
        n_page = n_seq
    shape = (n_layer, n_page, case["hkv"], page, case["dh"])
    dt = TYPES[case["type"]]
    st = dict(page=page, k=torch.randn(shape, generator=g, device="cuda").to(dt), v=torch.randn(shape, generator=g, device="cuda").to(dt),
              len=torch.tensor(held, dtype=torch.int32, device="cuda"), table=None, ref=None)
    if case["page"]:
        order = torch.randperm(n_page, generator=g, device="cuda")
        table = torch.full((n_seq, per), -1, dtype=torch.int32)
        used = torch.zeros(n_seq, per, dtype=torch.bool)
        for s, w in enumerate(want):
            used[s, :w] = True
        used = used.cuda()
        table = table.cuda()
        table[used] = order[:sum(want)].int()
        st["table"] = table
        st["ref"] = torch.zeros(n_page, dtype=torch.int32, device="cuda")
        st["ref"][order[:sum(want)]] = 1
    return st


def _runs(st, lens, past):
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    dev = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    st.update(lens=lens, past=past, starts=starts, rows=starts[-1], start=dev(starts), seq=dev(list(range(len(lens)))), pos=dev(past))


def _parents(lens, branch, g):
    """Each run a tree laid out level by level: node 0 the root, every node's parent among the `branch`-ary choices before it."""
    out = []
    for n in lens:
        pick = torch.rand(n, generator=g, device="cuda").cpu().tolist()
        for i in range(n):
            out.append(-1 if i == 0 else max(0, (i - 1) // branch - int(pick[i] * 2) * (i > 2 * branch)))
    return torch.tensor(out, dtype=torch.int32, device="cuda")


def _path(n, accept, g):
    """An accepted path through n nodes: the root, then nodes that lie either in their place already or behind the path."""
    a = min(accept, n)
    far = torch.randint(0, 1 << 30, (a,), generator=g, device="cuda").cpu().tolist()
    path = [0]
    for j in range(1, a):
        lo, hi = max(path[-1] + 1, a), n - (a - 1 - j)  # room for the rest of the path
        if lo >= hi:
            return list(range(a))
        path.append(lo + far[j] % min(hi - lo, 6))
    return path


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    op, lens = case["op"], _ints(case["lens"])
    randn = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    if op == "fork":
        n_par, ways = len(lens), case["ways"]
        held = lens + [0] * (n_par * ways)
        n_seq = len(held)
        st = _cache_for_fork(case, g, held) if case["page"] else _cache(case, g, case["layers"], n_seq, held)
        src = [p for p in range(n_par) for _ in range(ways)]
        dst = [n_par + i for i in range(n_par * ways)]
        dev = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        st.update(src=dev(src), dst=dev(dst), drop=dev([-1] * n_par + [0] * len(dst)),
                  grown=dev([-1] * n_par + [lens[p] + case["grow"] for p in src]), case=case, held=held, src_list=src, dst_list=dst)
        return st
    past = _ints(case["past"])
    ends = [a + b for a, b in zip(lens, past)]
    st = _cache(case, g, case.get("layers", 1), len(lens), ends)
    _runs(st, lens, past)
    st["case"] = case
    if op == "compact":
        paths = [_path(n, case["accept"], g) for n in lens]
        wide = max(len(p) for p in paths)
        st["paths"] = paths
        st["path"] = torch.tensor([p + [-1] * (wide - len(p)) for p in paths], dtype=torch.int32, device="cuda")
        st["n_path"] = torch.tensor([len(p) for p in paths], dtype=torch.int32, device="cuda")
        return st
    hq, hkv, dh, rows = case["hq"], case["hkv"], case["dh"], st["rows"]
    if op == "prep":
        sec = _ints(case["sections"])
        half = case["n_rot"] // 2
        axis = [i for i, n in enumerate(sec) for _ in range(n)]
        if case["mixed"]:  # dealt out in turn while an axis has pairs left
            left, axis = list(sec), []
            while len(axis) < half:
                for i in range(len(sec)):
                    if left[i]:
                        left[i] -= 1
                        axis.append(i)
        st["pair_axis"] = torch.tensor(axis, dtype=torch.uint8, device="cuda")
        st["q"] = 2 * randn(rows, hq, (2 if case["gated"] else 1) * dh)
        st["kin"], st["vin"] = 3 * randn(rows, hkv, dh), randn(rows, hkv, dh)
        st["qn"], st["kn"] = 1 + 0.2 * randn(dh), 1 + 0.2 * randn(dh)
        t = torch.cat([torch.arange(p, p + n, device="cuda") for n, p in zip(lens, past)])
        hw = torch.randint(0, 64, (2, rows), generator=g, device="cuda")
        image = torch.rand(rows, generator=g, device="cuda") < 0.5  # rows of an image keep one time step and have a height and width of their own
        st["axis_pos"] = torch.stack([t - t % 7 * image] + [torch.where(image, (t - t % 7 + hw[i]).clamp(max=case["cap"] - 1), t) for i in range(2)]).int().contiguous()
        ang = torch.arange(case["cap"], device="cuda", dtype=torch.float64)[:, None] * 1e7 ** (-2.0 * torch.arange(half, device="cuda", dtype=torch.float64) / case["n_rot"])
        st["rope"] = torch.stack([ang.cos(), ang.sin()], dim=-1).float().contiguous()
        return st
    st["q"] = 1.5 * randn(rows, hq, dh)
    st["qfull"] = randn(rows, hq, 2 * dh) if case["gated"] else None
    if op == "tree":
        st["parent"] = _parents(lens, case["branch"], g)
    return st


def _cache_for_fork(case, g, held):
    """Pages for the parents and for what their children will take beside the shared ones."""
    page, ways, n = case["page"], case["ways"], sum(1 for h in held if h)
    more = sum((-(-(h + case["grow"]) // page) - h // page) * ways for h in held[:n])
    st = _cache(case, g, case["layers"], len(held), held)
    lack = more - int((st["ref"] == 0).sum())
    if lack > 0:
        shape = list(st["k"].shape)
        shape[1] = lack
        add = lambda t: torch.cat([t, torch.randn(shape, generator=g, device="cuda").to(t.dtype)], dim=1).contiguous()  # noqa: E731
        st["k"], st["v"] = add(st["k"]), add(st["v"])
        st["ref"] = torch.cat([st["ref"], torch.zeros(lack, dtype=torch.int32, device="cuda")])
    return st


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(state):
    if own:
        return _own(state)
    return {"prep": _prep, "packed": _packed, "tree": _tree, "fork": _fork, "compact": _compact}[state["case"]["op"]](state)


def _own(st):
    """The calls a user makes of the library; the handles and workspaces are made once, as such a program keeps them."""
    import __graft_entry__
    qk = __graft_entry__.load_package()
    op = st["case"]["op"]
    if "handle" not in st:
        st["handle"] = cache = qk.KvCache(st["k"], st["v"], table=st["table"], ref=st["ref"], len=st["len"])
        if op in ("prep", "packed", "tree"):
            st["batch"] = qk.KvRuns(st["rows"], st["start"], st["seq"], st["pos"], max_run=max(st["lens"]))
        if op in ("packed", "tree"):
            st["ws"] = torch.empty(qk.attn_runs_workspace_bytes(cache, st["batch"], st["case"]["hq"]), dtype=torch.uint8, device="cuda")
        if op == "fork":
            st["ws"] = torch.empty(qk.kv_workspace_bytes(cache), dtype=torch.uint8, device="cuda")
    cache = st["handle"]
    if op == "prep":
        qhat = qk.attn_prep_axes(cache, 0, st["batch"], st["q"], st["kin"], st["vin"], st["qn"], st["kn"], st["rope"], st["pair_axis"],
                                 st["axis_pos"], eps=EPS)
        return dict(qhat=qhat, k=st["k"], v=st["v"])
    if op == "packed":
        return qk.attn_packed(cache, 0, st["batch"], st["q"], st["ws"], qfull=st["qfull"])
    if op == "tree":
        return qk.attn_tree(cache, 0, st["batch"], st["parent"], st["q"], st["ws"], qfull=st["qfull"])
    if op == "compact":
        qk.kv_compact(cache, st["seq"], st["pos"], st["path"], st["n_path"])
        return dict(k=st["k"], v=st["v"])
    a = qk.kv_resize(cache, st["drop"], st["ws"])
    b = qk.kv_fork(cache, st["src"], st["dst"], st["ws"])
    c = qk.kv_resize(cache, st["grown"], st["ws"])
    return _books(st, a, b, c)


def _books(st, *status):
    out = dict(k=st["k"], v=st["v"], len=st["len"], status=status)
    if st["table"] is not None:
        out.update(table=st["table"], ref=st["ref"])
    return out


def _place(st, row_seq, row_pos):
    """(page, row in it) of cache rows."""
    if st["table"] is None:
        return row_seq, row_pos
    return st["table"][row_seq, row_pos // st["page"]].long(), row_pos % st["page"]


def _prep(st):
    c = st["case"]
    rows, dh, half = st["rows"], c["dh"], c["n_rot"] // 2
    i = torch.arange(rows, device="cuda")
    run_of = torch.searchsorted(st["start"].long(), i, right=True) - 1
    pos = st["pos"].long()[run_of] + i - st["start"].long()[run_of]
    ang = st["rope"][st["axis_pos"].long()[st["pair_axis"].long()].t(), torch.arange(half, device="cuda")]  # [rows, half, 2]
    cos, sin = ang[:, None, :, 0], ang[:, None, :, 1]

    def turn(x, w):
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        a, b = x[..., :half], x[..., half:2 * half]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., 2 * half:]], dim=-1)

    page, row = _place(st, st["seq"].long()[run_of], pos)
    st["k"][0, page, :, row] = turn(st["kin"], st["kn"]).to(st["k"].dtype)
    st["v"][0, page, :, row] = st["vin"].to(st["v"].dtype)
    return dict(qhat=turn(st["q"][..., :dh], st["qn"]), k=st["k"], v=st["v"])


def _rows_of(st, pool, seq, n):
    """Cache rows 0 .. n of sequence seq, [hkv, n, dh] in 32 bits."""
    if st["table"] is None:
        return pool[0, seq, :, :n].float()
    pages = st["table"][seq, :-(-n // st["page"])].long()
    x = pool[0, pages].transpose(0, 1)  # [hkv, pages, rows, dh]
    return x.reshape(x.shape[0], -1, x.shape[-1])[:, :n].float()


def _gate(st, att):
    return att if st["qfull"] is None else att * torch.sigmoid(st["qfull"][..., att.shape[-1]:])


def _packed(st):
    c = st["case"]
    hq, hkv, dh = c["hq"], c["hkv"], c["dh"]
    group = hq // hkv
    att = torch.empty_like(st["q"])
    for s, (n, past) in enumerate(zip(st["lens"], st["past"])):
        lo, total = st["starts"][s], past + n
        k, v = _rows_of(st, st["k"], s, total), _rows_of(st, st["v"], s, total)
        q = st["q"][lo:lo + n].view(n, hkv, group, dh).permute(1, 2, 0, 3).reshape(hkv, group * n, dh)
        score = (torch.matmul(q, k.transpose(1, 2)) / math.sqrt(dh)).view(hkv, group, n, total)
        later = torch.arange(total, device="cuda") > past + torch.arange(n, device="cuda")[:, None]
        p = torch.softmax(score.masked_fill_(later, -math.inf), dim=-1)
        o = torch.matmul(p.view(hkv, group * n, total), v)
        att[lo:lo + n] = o.view(hkv, group, n, dh).permute(2, 0, 1, 3).reshape(n, hq, dh)
    return _gate(st, att)


def _family(st):
    """[rows, rows] of ancestors and self, by doubling: who is reached in up to 1, 2, 4, ... steps to the parent."""
    rows = st["rows"]
    i = torch.arange(rows, device="cuda")
    run_of = torch.searchsorted(st["start"].long(), i, right=True) - 1
    up = torch.where(st["parent"] < 0, i, st["parent"].long() + st["start"].long()[run_of])
    kin = (i[:, None] == i) | (up[:, None] == i)
    return _doubled(kin.float(), max(st["lens"]))


def _doubled(kin, n):
    step = 1
    while step < n:
        kin = (torch.matmul(kin, kin) > 0).float()
        step *= 2
    return kin > 0


def _tree(st):
    c = st["case"]
    hq, hkv, dh, n_run = c["hq"], c["hkv"], c["dh"], len(st["lens"])
    group, wide, top = hq // hkv, max(st["lens"]), max(a + b for a, b in zip(st["lens"], st["past"]))
    slot = st["start"].long()[:-1, None] + torch.arange(wide, device="cuda")  # row of (run, node); past a run's end: of another run, dropped below
    slot = slot.clamp(max=st["rows"] - 1)
    kin = _family(st)[slot[:, :, None], slot[:, None, :]]  # [run, node, node]
    key = torch.arange(top, device="cuda")
    node = key - st["pos"].long()[:, None]  # [run, top]: which node a key is, negative: a cached row
    seen = torch.gather(kin, 2, node.clamp(0, wide - 1)[:, None, :].expand(n_run, wide, top))
    count = (st["start"][1:] - st["start"][:-1]).long()[:, None, None]
    seen = ((node[:, None, :] < 0) | seen) & (node[:, None, :] < count)
    if st["table"] is None:
        k, v = st["k"][0, st["seq"].long(), :, :top].float(), st["v"][0, st["seq"].long(), :, :top].float()
    else:
        pages = st["table"][st["seq"].long(), :-(-top // st["page"])].long().clamp(min=0)
        k, v = (x[0, pages].transpose(1, 2).reshape(n_run, hkv, -1, dh)[:, :, :top].float() for x in (st["k"], st["v"]))
    q = st["q"][slot].view(n_run, wide, hkv, group, dh).permute(0, 2, 3, 1, 4).reshape(n_run, hkv, group * wide, dh)
    score = (torch.matmul(q, k.transpose(2, 3)) / math.sqrt(dh)).view(n_run, hkv, group, wide, top)
    p = torch.softmax(score.masked_fill(~seen[:, None, None], -1e30), dim=-1)
    o = torch.matmul(p.view(n_run, hkv, group * wide, top), v).view(n_run, hkv, group, wide, dh).permute(0, 3, 1, 2, 4).reshape(n_run, wide, hq, dh)
    i = torch.arange(st["rows"], device="cuda")
    run_of = torch.searchsorted(st["start"].long(), i, right=True) - 1
    return _gate(st, o[run_of, i - st["start"].long()[run_of]])


def _resize(st, new, grows):
    """Lengths `new` (-1: unchanged; not `grows`: none is longer than before): pages behind the end given back, missing ones taken lowest first, a shared part-filled page
    replaced by a copy before its sequence grows."""
    ln, page = st["len"], st["page"]
    if st["table"] is None:
        ln.copy_(torch.where(new < 0, ln, new))
        return torch.zeros(1, dtype=torch.int32, device="cuda")
    table, ref = st["table"], st["ref"]
    n_seq, per = table.shape
    n_page = ref.shape[0]
    new = torch.where(new < 0, ln, new).long()
    old = ln.long()
    want, have = -(-new // page), -(-old // page)
    col = torch.arange(per, device="cuda")
    gone = (col >= want[:, None]) & (col < have[:, None])
    ref.index_add_(0, table.clamp(min=0).long().view(-1), -gone.view(-1).int())
    table.masked_fill_(gone, -1)
    last = (old - 1).clamp(min=0) // page
    last_page = table.gather(1, last[:, None])[:, 0].long().clamp(min=0)
    split = (new > old) & (old % page != 0) & (ref[last_page] > 1)
    need = (want - have).clamp(min=0) + split
    free = ref == 0
    missing = (need.sum() - free.sum()).clamp(min=0)
    fits = missing == 0
    need, split = need * fits, split & fits
    order = torch.argsort(free.int(), descending=True, stable=True)  # free pages first, lowest first
    first = need.cumsum(0) - need
    fresh = ((col >= have[:, None]) & (col < want[:, None]) & fits) | (split[:, None] & (col == last[:, None]))
    place = first[:, None] + fresh.long().cumsum(1) - 1
    taken = order[place.clamp(0, n_page - 1)]
    to_page = torch.where(split, taken.gather(1, last[:, None])[:, 0], last_page)
    table.copy_(torch.where(fresh, taken.int(), table))
    ref.index_add_(0, taken.view(-1), fresh.view(-1).int())
    ref.index_add_(0, last_page, -split.int())
    keep = (torch.arange(page, device="cuda") < (old % page)[:, None]) & split[:, None]  # [seq, row]
    if grows:  # a sequence without a copy to make writes its last page onto itself
        for pool in (st["k"], st["v"]):
            pool[:, to_page] = torch.where(keep[None, :, None, :, None], pool[:, last_page], pool[:, to_page])
    ln.copy_(torch.where((new > old) & ~fits, old, new).int())
    return missing.int().view(1)


def _fork(st):
    a = _resize(st, st["drop"], False)
    src, dst = st["src"].long(), st["dst"].long()
    if st["table"] is None:
        row = torch.arange(st["page"], device="cuda") < st["len"][src][:, None]
        for pool in (st["k"], st["v"]):
            pool[:, dst] = torch.where(row[None, :, None, :, None], pool[:, src], pool[:, dst])
    else:
        st["table"][dst] = st["table"][src]
        st["ref"].index_add_(0, st["table"][src].clamp(min=0).long().view(-1), (st["table"][src] >= 0).view(-1).int())
    st["len"][dst] = st["len"][src]
    b = torch.zeros(1, dtype=torch.int32, device="cuda")
    return _books(st, a, b, _resize(st, st["grown"], True))


def _compact(st):
    path, count = st["path"].long(), st["n_path"].long()
    n, wide = path.shape
    j = torch.arange(wide, device="cuda").expand(n, wide)
    path = torch.where(j < count[:, None], path, j)  # behind the path: a row onto itself
    seq = st["seq"].long()[:, None].expand(n, wide)
    last = (st["pos"] + (st["start"][1:] - st["start"][:-1])).long()[:, None] - 1
    from_page, from_row = _place(st, seq, (st["pos"].long()[:, None] + path).minimum(last))
    to_page, to_row = _place(st, seq, (st["pos"].long()[:, None] + j).minimum(last))
    for pool in (st["k"], st["v"]):
        pool[:, to_page, :, to_row] = pool[:, from_page, :, from_row]
    return dict(k=st["k"], v=st["v"])


# ---- what a pass cannot do without ------------------------------------------------------------------------------------

def work(case):
    lens = _ints(case["lens"])
    size = 4 if case["type"] == "f32" else 2
    dh, hkv = case["dh"], case["hkv"]
    op = case["op"]
    if op == "fork":
        page = case["page"] or case["cap"]
        rows = sum(n % page if case["page"] else n for n in lens) * case["ways"]
        return dict(bytes=2 * 2 * rows * case["layers"] * hkv * dh * size + 8 * len(lens) * case["cap"] // page, flops=0)
    past = _ints(case["past"])
    if op == "compact":
        rows = sum(max(0, min(case["accept"], n) - 1) for n in lens)
        return dict(bytes=2 * 2 * rows * case["layers"] * hkv * dh * size, flops=0)
    rows, hq = sum(lens), case["hq"]
    if op == "prep":
        return dict(bytes=rows * (2 * hq * dh * 4 + 2 * hkv * dh * (4 + size) + 12 + 8 * case["n_rot"] // 2), flops=rows * (hq + hkv) * dh * 8)
    keys = sum(n + p for n, p in zip(lens, past))
    pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(lens, past))
    if op == "tree":  # a node sees the cached rows and its ancestors: here about log(n) of the nodes, at most all
        pairs = sum(n * (p + 1 + int(math.log2(n + 1))) for n, p in zip(lens, past))
    gate = rows * hq * dh * 4 if case["gated"] else 0
    return dict(bytes=2 * rows * hq * dh * 4 + gate + 2 * keys * hkv * dh * size, flops=4 * dh * hq * pairs)


# ---- the same in 64 bits, from the definitions -------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "fork":
        return _exact_fork(st)
    page_of = (lambda s, r: (s, r)) if st["table"] is None else (lambda s, r, t=st["table"].tolist(), n=st["page"]: (t[s][r // n], r % n))
    if op == "compact":
        k, v = st["k"].double(), st["v"].double()
        for s, path in enumerate(st["paths"]):
            base = st["past"][s]
            moved = [[pool[:, page_of(s, base + i)[0], :, page_of(s, base + i)[1]].clone() for i in path] for pool in (k, v)]
            for pool, rows in zip((k, v), moved):
                for j, r in enumerate(rows):
                    at = page_of(s, base + j)
                    pool[:, at[0], :, at[1]] = r
        return dict(k=k, v=v)
    dh, hq, hkv = case["dh"], case["hq"], case["hkv"]
    if op == "prep":
        half = case["n_rot"] // 2
        where = [page_of(s, st["past"][s] + i) for s, n in enumerate(st["lens"]) for i in range(n)]
        pages, rows = (torch.tensor([w[i] for w in where], device="cuda") for i in (0, 1))
        at = st["axis_pos"].long().index_select(0, st["pair_axis"].long())  # [half, rows]
        z = torch.view_as_complex(st["rope"].double().contiguous())  # cos + i sin
        z = torch.stack([z[at[j], j] for j in range(half)], dim=1)[:, None, :]

        def turned(x, w):
            x = x.double()
            x = x / (x.square().sum(-1, keepdim=True) / dh + EPS).sqrt() * w.double()
            pair = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * z
            return torch.cat([pair.real, pair.imag, x[..., 2 * half:]], dim=-1)

        k, v = st["k"].double(), st["v"].double()
        k[0, pages, :, rows] = turned(st["kin"], st["kn"])
        v[0, pages, :, rows] = st["vin"].double()
        return dict(qhat=turned(st["q"][..., :dh], st["qn"]), k=k, v=v)
    out = torch.zeros(st["rows"], hq, dh, dtype=torch.float64, device="cuda")
    parent = st["parent"].tolist() if op == "tree" else None
    for s, (n, past) in enumerate(zip(st["lens"], st["past"])):
        total, lo = past + n, st["starts"][s]
        see = torch.zeros(n, total, dtype=torch.bool)
        see[:, :past] = True
        for i in range(n):
            if op == "packed":
                see[i, past:past + i + 1] = True
            else:
                a = i
                while a >= 0:
                    see[i, past + a] = True
                    a = parent[lo + a]
        see = see.cuda()
        pages = [st["table"][s].tolist()[b] for b in range(-(-total // st["page"]))] if st["table"] is not None else [s]
        for h in range(hq):
            kk = torch.cat([st["k"][0, p, h // (hq // hkv)] for p in pages])[:total].double()
            vv = torch.cat([st["v"][0, p, h // (hq // hkv)] for p in pages])[:total].double()
            score = st["q"][lo:lo + n, h].double() @ kk.t() * dh ** -0.5
            score[~see] = -math.inf
            w = (score - score.max(dim=1, keepdim=True).values).exp()
            out[lo:lo + n, h] = (w @ vv) / w.sum(dim=1, keepdim=True)
    if st["qfull"] is not None:
        out = out / (1 + (-st["qfull"][..., dh:].double()).exp())
    return out


def _exact_fork(st):
    """The books kept one sequence after the other with plain lists."""
    page = st["page"]
    k, v = st["k"].double(), st["v"].double()
    ln, grown = list(st["held"]), st["grown"].tolist()
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    if st["table"] is None:
        for s, d in zip(st["src_list"], st["dst_list"]):
            for pool in (k, v):
                pool[:, d, :, :ln[s]] = pool[:, s, :, :ln[s]]
        ln = [g if g >= 0 else n for g, n in zip(grown, ln)]
        return dict(k=k, v=v, len=ints(ln), status=(ints([0]),) * 3)
    table, ref = st["table"].tolist(), st["ref"].tolist()
    per = len(table[0])
    for s, d in zip(st["src_list"], st["dst_list"]):
        ln[d] = ln[s]
        table[d] = list(table[s])
        for p in table[s]:
            if p >= 0:
                ref[p] += 1
    free = [p for p, r in enumerate(ref) if r == 0]
    shared = [r > 1 for r in ref]
    for s, want in enumerate(grown):
        if want < 0:
            continue
        rest = ln[s] % page
        if rest and shared[table[s][ln[s] // page]]:
            old, fresh = table[s][ln[s] // page], free.pop(0)
            for pool in (k, v):
                pool[:, fresh, :, :rest] = pool[:, old, :, :rest]
            ref[old] -= 1
            ref[fresh] = 1
            table[s][ln[s] // page] = fresh
        for b in range(-(-ln[s] // page), -(-want // page)):
            table[s][b] = free.pop(0)
            ref[table[s][b]] = 1
        ln[s] = want
    assert all(len(t) == per for t in table)
    return dict(k=k, v=v, len=ints(ln), status=(ints([0]),) * 3, table=ints(table), ref=ints(ref))
