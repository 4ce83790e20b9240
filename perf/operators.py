"""The operators of serving many sequences from one paged KV cache, with their plain forms.

Three operators, each over the range of sizes a server meets:

  attend  decode attention of one new token for every row of a batch over the paged cache, the new
          token's key and value stored by the same call (moearc_b200.kvcache.KvCache.attn_decode)
  refork, rollback, compact
          the cache's pages: rows dropped and forked again from a kept row, rows cut back and grown
          (a speculative step's rejected tokens), live pages moved together
          (KvCache.free / fork / grow / compact)
  score   log probabilities of given tokens under rows of logits, with the distribution's entropy
          and its k likeliest tokens (Context.token_logprobs)

Page tables, lengths and reference counts are int32 tensors; a table entry of -1 is no page.
"""
import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GGUF = {"f32": 0, "f16": 1, "bf16": 30}
DEV = "cuda"


# ---- the cases ---------------------------------------------------------------------------------

def listed():
    return [
        # one stream early in its context, the decoder's own head layout: latency only
        dict(name="attend_one", op="attend", rows=1, pad=0, max_kv=257, heads=64, kv_heads=8, dim=64, kv="bf16", page=32,
             window=0, sinks=True, append=True),
        # a window layer of the same layout under a batch with padded rows: short spans of long contexts
        dict(name="attend_window", op="attend", rows=120, pad=8, max_kv=8000, heads=64, kv_heads=8, dim=64, kv="bf16", page=32,
             window=128, sinks=True, append=True),
        # the batched decoder's 64 streams at depth 4096, ragged
        dict(name="attend_streams", op="attend", rows=64, pad=0, max_kv=4096, heads=32, kv_heads=4, dim=128, kv="bf16", page=32,
             window=0, sinks=False, append=True),
        # few long contexts: the split over the length carries it
        dict(name="attend_long", op="attend", rows=3, pad=0, max_kv=100001, heads=32, kv_heads=8, dim=128, kv="f16", page=64,
             window=0, sinks=False, append=True),
        # an f32 cache with odd head sizes and a page size that divides nothing
        dict(name="attend_f32", op="attend", rows=21, pad=1, max_kv=2999, heads=20, kv_heads=5, dim=80, kv="f32", page=17,
             window=0, sinks=True, append=False),
        # beams of one small model: the losing beams dropped, the winners forked over their rows
        dict(name="refork_beams", op="refork", rows=16, parents=3, max_kv=700, layers=2, pages=1024, kv_heads=4, dim=64, kv="f16",
             page=16, deep=False),
        # whole copies of prompts for rows that will be changed in place, every layer
        dict(name="refork_deep", op="refork", rows=40, parents=8, max_kv=900, layers=36, pages=2000, kv_heads=8, dim=64,
             kv="bf16", page=32, deep=True),
        # a speculative step over a serving batch: rejected tokens cut off, rows grown for the next draft
        dict(name="rollback_batch", op="rollback", rows=256, max_kv=4000, draft=6, layers=8, pages=40000, kv_heads=4, dim=64,
             kv="bf16", page=16),
        # a fragmented pool moved together so that its tail can be given back
        dict(name="compact_pool", op="compact", rows=60, max_kv=2000, live=0.5, layers=12, pages=6001, kv_heads=8, dim=64,
             kv="bf16", page=32),
        # one stream's next-token logits
        dict(name="score_one", op="score", rows=1, vocab=131072, stride=131072, type="f32", k=8, masked=0.0, scale=1.0),
        # a decode batch over a large vocabulary, a grammar's mask, rows inside a wider buffer
        dict(name="score_batch", op="score", rows=64, vocab=200019, stride=200064, type="f32", k=20, masked=0.4, scale=1.25),
        # a prompt scored token by token from bf16 logits
        dict(name="score_prompt", op="score", rows=2047, vocab=100003, stride=100003, type="bf16", k=5, masked=0.0, scale=1.0),
    ]


HEADS = ((64, 8, 64), (32, 4, 128), (32, 8, 128), (20, 5, 80), (8, 8, 64), (48, 3, 128), (16, 1, 256), (12, 2, 96), (7, 7, 72))
MOST_BYTES = 1.0e9  # of a drawn case; the largest listed one has more


def _log(rng, lo, hi):
    return int(round(float(np.exp(rng.uniform(np.log(lo), np.log(hi))))))


def draw(rng):
    op = rng.choice(("attend", "attend", "attend", "refork", "rollback", "compact", "score", "score"))
    kv = rng.choice(("bf16", "bf16", "f16", "f32"))
    page = rng.choice((1, 8, 16, 17, 32, 64, _log(rng, 2, 128)))
    if op == "attend":
        heads, kv_heads, dim = rng.choice(HEADS)
        case = dict(op=op, rows=_log(rng, 1, 300), pad=rng.choice((0, 0, 1, 5)), max_kv=_log(rng, 1, 60000), heads=heads, kv_heads=kv_heads,
                    dim=dim, kv=kv, page=page, window=rng.choice((0, 0, 0, 128, _log(rng, 1, 4000))), sinks=rng.random() < 0.5,
                    append=rng.random() < 0.7)
    elif op == "score":
        vocab = _log(rng, 900, 250000)
        case = dict(op=op, rows=_log(rng, 1, 3000), vocab=vocab, stride=vocab + rng.choice((0, 0, 1, 61)), type=rng.choice(("f32", "f32", "bf16", "f16")),
                    k=rng.choice((0, 1, 5, 20, 32)), masked=rng.choice((0.0, 0.0, 0.3, 0.99)), scale=rng.choice((1.0, 1.0, 0.5, 1.4)))
    else:
        kv_heads, dim = rng.choice(((8, 64), (4, 128), (5, 80), (1, 256)))
        case = dict(op=op, rows=_log(rng, 2, 200), max_kv=_log(rng, 2, 3000), layers=_log(rng, 1, 24), kv_heads=kv_heads, dim=dim, kv=kv,
                    page=max(4, page))
        if op == "refork":
            case.update(deep=rng.random() < 0.4, parents=_log(rng, 1, max(1, case["rows"] // 2)))
        elif op == "rollback":
            case.update(draft=_log(rng, 1, 40))
        else:
            case.update(live=rng.choice((0.2, 0.5, 0.9)))
    while True:
        if op in ("refork", "rollback", "compact"):  # a pool that holds what the case needs
            most = case["rows"] * (-(-(case["max_kv"] + case.get("draft", 0)) // case["page"]) + 1)
            case["pages"] = int(most * (2.1 if op != "compact" else 1 / case["live"])) + 7
            size = 2 * case["layers"] * case["pages"] * _page_bytes(case)
        else:
            size = 0
        if work(case)["bytes"] <= MOST_BYTES and size <= 6e9:
            return case
        big = "max_kv" if op != "score" and case["max_kv"] > 8 * case["page"] else "rows"
        case[big] = max(1, case[big] // 2)
        if op == "refork":
            case["rows"] = max(2, case["rows"])
            case["parents"] = max(1, min(case["parents"], case["rows"] // 2))
        if big == "rows" and case["rows"] <= 2 and op != "score":
            case["max_kv"] = max(1, case["max_kv"] // 2)
            case["layers"] = max(1, case.get("layers", 1) // 2)


def _page_bytes(case):
    return case["page"] * case["kv_heads"] * case["dim"] * torch.empty(0, dtype=TYPES[case["kv"]]).element_size()


def _rs(case):
    """Lengths and layouts go by the case alone, so that work() knows them; values go by the seed."""
    return np.random.RandomState(sum(ord(c) * (i + 1) for i, c in enumerate(case["op"])) + 7 * case["rows"] + case["max_kv"])


def _lengths(case):
    """Ragged lengths up to max_kv, one row at the most, every padded row empty."""
    n = case["rows"]
    got = _rs(case).randint(max(1, case["max_kv"] // 3), case["max_kv"] + 1, n)
    got[n // 2] = case["max_kv"]
    pad = min(case.get("pad", 0), n - 1)
    if pad:
        got[_rs(case).permutation(np.delete(np.arange(n), n // 2))[:pad]] = 0
    return got.astype(np.int64)


def _begins(case, n_kv):
    return np.maximum(n_kv - case["window"], 0) if case["window"] else np.zeros_like(n_kv)


def _pages_of(n_kv, page):
    return -(-n_kv // page)


def _parents(case):
    """The row that each row is forked from: rows 0 .. parents - 1 are kept, the others are children."""
    return np.arange(case["rows"] - case["parents"]) % case["parents"]


def work(case):
    op = case["op"]
    if op == "score":
        size = torch.empty(0, dtype=TYPES[case["type"]]).element_size()
        cells = case["rows"] * case["vocab"]
        return {"bytes": cells * size + case["rows"] * (12 + 8 * case["k"]), "flops": 6 * cells}
    n_kv = _lengths(case)
    if op == "attend":
        size = torch.empty(0, dtype=TYPES[case["kv"]]).element_size()
        keys = int((n_kv - _begins(case, n_kv)).sum())
        row = case["kv_heads"] * case["dim"] * size
        fresh = case["rows"] * 2 * case["kv_heads"] * case["dim"] * (4 + size) if case["append"] else 0
        return {"bytes": 2 * keys * row + 8 * case["rows"] * case["heads"] * case["dim"] + fresh,
                "flops": 4 * keys * case["heads"] * case["dim"]}
    tables = 4 * int(_pages_of(n_kv, case["page"]).sum())
    if op == "refork":
        p, kept = _parents(case), n_kv[: case["parents"]]
        moved = int(_pages_of(kept[p], case["page"]).sum()) if case["deep"] else int((kept[p] % case["page"] != 0).sum())
    elif op == "rollback":
        moved = 0  # a shared last page is copied once, when a row is first grown over it
    else:
        moved = int(_pages_of(n_kv, case["page"]).sum() * (1 - case["live"]))
    return {"bytes": 4 * case["layers"] * moved * _page_bytes(case) + 2 * tables + 4 * case["pages"], "flops": 0}


def _kept(case, n_kv):
    """What a verified draft leaves of each row."""
    return np.maximum(n_kv - _rs(case).randint(0, case["draft"] + 1, len(n_kv)), 1)


# ---- their inputs ------------------------------------------------------------------------------

def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(DEV)


def _rows_to_tables(case, n_kv, ids, stride):
    """Page tables with the pages `ids` handed out row by row."""
    tables = np.full((len(n_kv), stride), -1, np.int64)
    at = 0
    for s, n in enumerate(_pages_of(n_kv, case["page"])):
        tables[s, :n] = ids[at:at + n]
        at += n
    return tables, at


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    st = dict(case=case)
    if case["op"] == "score":
        dt = TYPES[case["type"]]
        x = torch.randn(case["rows"], case["stride"], generator=g, device=DEV, dtype=torch.float32) * 2.5
        if case["masked"]:  # a grammar's mask: the same cut of the vocabulary for a row and its neighbours
            hide = torch.rand(case["rows"], case["stride"], generator=g, device=DEV) < case["masked"]
            x[hide] = -torch.inf
        st["logits"] = x.to(dt)
        st["tokens"] = torch.randint(0, case["vocab"], (case["rows"],), generator=g, device=DEV, dtype=torch.int32)
        st["logprob"], st["entropy"] = (torch.empty(case["rows"], device=DEV) for _ in range(2))
        st["top_ids"] = torch.empty(case["rows"], case["k"], device=DEV, dtype=torch.int32)
        st["top_logprobs"] = torch.empty(case["rows"], case["k"], device=DEV)
        torch.cuda.synchronize()
        return st
    rs, n_kv, page = np.random.RandomState(seed % (1 << 31)), _lengths(case), case["page"]
    dt, op, layers = TYPES[case["kv"]], case["op"], case.get("layers", 1)
    need = _pages_of(n_kv + case.get("draft", 0), page)
    stride = int(need.max()) + 3
    if op == "attend":
        pages = int(need.sum()) + 5
        tables, _ = _rows_to_tables(case, n_kv, rs.permutation(pages), stride)
        begin = _begins(case, n_kv)
        H, D = case["heads"], case["dim"]
        st["span"] = int((n_kv - begin).max())
        st["begin"] = _i32(begin) if case["window"] else None
        row = (H + 2 * case["kv_heads"]) * D  # q, k and v of a row as one projection leaves them
        st["qkv"] = torch.randn(case["rows"], row, generator=g, device=DEV)
        st["sinks"] = torch.randn(H, generator=g, device=DEV) if case["sinks"] else None
        st["out"] = torch.empty(case["rows"], H, D, device=DEV)
        refs = np.bincount(tables[tables >= 0], minlength=pages)
    else:
        pages = case["pages"]
        if op == "refork":  # parents hold their pages; each child still shares a parent's, from an earlier fork
            kept, p = n_kv[: case["parents"]], _parents(case)
            tables = np.full((case["rows"], stride), -1, np.int64)
            ids = rs.permutation(pages)
            tables[: case["parents"]], at = _rows_to_tables(case, kept, ids, stride)
            old = np.minimum(kept[(p + 1) % case["parents"]], n_kv[case["parents"]:])
            for c, n in enumerate(old):
                full = n // page
                tables[case["parents"] + c, :full] = tables[(p[c] + 1) % case["parents"], :full]
                if n % page:
                    tables[case["parents"] + c, full] = ids[at]
                    at += 1
            n_kv = np.concatenate([kept, old])
            st["src"], st["dst"] = [int(v) for v in p], list(range(case["parents"], case["rows"]))
        else:
            ids = rs.permutation(pages)
            if op == "rollback":  # every fourth row was forked from the row before it and shares its pages
                twin = np.arange(3, case["rows"], 4)
                kept = _kept(case, n_kv)
                n_kv[twin], kept[twin] = n_kv[twin - 1], kept[twin - 1]
                mine = n_kv.copy()
                mine[twin] = 0
                tables, _ = _rows_to_tables(case, mine, ids, stride)
                tables[twin] = tables[twin - 1]
                st["rows"], st["keep"], st["add"] = list(range(case["rows"])), [int(v) for v in kept], [case["draft"]] * case["rows"]
            else:
                need = int(_pages_of(n_kv, page).sum())
                spread = rs.permutation(min(pages, max(need, int(need / case["live"]))))
                tables, _ = _rows_to_tables(case, n_kv, spread, stride)
        refs = np.bincount(tables[tables >= 0], minlength=pages)
        st["tables_out"] = torch.empty(tables.shape, device=DEV, dtype=torch.int32)
        st["refs_out"] = torch.empty(pages, device=DEV, dtype=torch.int32)
        st["n_live"] = torch.empty(1, device=DEV, dtype=torch.int32)
    shape = (layers, pages, page, case["kv_heads"], case["dim"])
    st["k"], st["v"] = (torch.randn(shape, generator=g, device=DEV, dtype=dt) for _ in range(2))
    st["tables"], st["n_kv"], st["refs"] = _i32(tables), _i32(n_kv), _i32(refs)
    torch.cuda.synchronize()  # the library's context has a stream of its own
    return st


# ---- the plain forms ---------------------------------------------------------------------------

def _attend(st):
    c = st["case"]
    H, G, D, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    q, kn, vn = st["qkv"].split([H * D, G * D, G * D], 1)
    k, v = st["k"][0].view(-1, G, D), st["v"][0].view(-1, G, D)
    tables, n_kv = st["tables"].long(), st["n_kv"].long()
    if c["append"]:  # the new token is the last of its row
        rows = torch.nonzero(n_kv > 0)[:, 0]
        last = n_kv[rows] - 1
        slot = tables[rows, last // page] * page + last % page
        k[slot], v[slot] = kn[rows].view(-1, G, D).to(k.dtype), vn[rows].view(-1, G, D).to(v.dtype)
    begin = st["begin"].long() if st["begin"] is not None else torch.zeros_like(n_kv)
    pos = begin[:, None] + torch.arange(st["span"], device=DEV)
    live = pos < n_kv[:, None]
    at = tables.gather(1, (pos // page).clamp(max=tables.shape[1] - 1))
    live &= at >= 0
    slot = torch.where(live, at * page + pos % page, 0)
    ks = k[slot].float()
    vs = torch.where(live[:, :, None, None], v[slot].float(), 0.0)
    x = torch.einsum("bgud,blgd->bgul", q.reshape(-1, G, H // G, D), ks) / D ** 0.5
    x = torch.where(live[:, None, None, :], x, -torch.inf)
    top = x.amax(-1, keepdim=True)
    if c["sinks"]:
        sink = st["sinks"].view(1, G, H // G, 1)
        top = torch.maximum(top, sink)
    top = torch.where(top == -torch.inf, 0.0, top)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    if c["sinks"]:
        total = total + torch.exp(sink - top)
    y = torch.einsum("bgul,blgd->bgud", e, vs) / torch.where(total == 0, 1.0, total)
    st["out"].copy_(y.reshape(-1, H, D))
    return {"out": st["out"], "k": st["k"], "v": st["v"]}


def _free(st, rows, keep):
    page, rows = st["case"]["page"], torch.tensor(rows, device=DEV)
    keep = torch.minimum(st["n_kv"][rows], torch.tensor(keep, device=DEV, dtype=torch.int32))
    have = st["tables"][rows]
    gone = (torch.arange(have.shape[1], device=DEV) >= -(-keep // page)[:, None]) & (have >= 0)
    drop = have[gone]
    st["refs"].index_add_(0, drop, torch.full_like(drop, -1))
    st["tables"][rows] = torch.where(gone, -1, have)
    st["n_kv"][rows] = keep


def _copy(st, src, dst):
    st["k"][:, dst] = st["k"][:, src]
    st["v"][:, dst] = st["v"][:, src]


def _fork(st, src, dst, deep):
    page, src, dst = st["case"]["page"], torch.tensor(src, device=DEV), torch.tensor(dst, device=DEV)
    have, n = st["tables"][src], st["n_kv"][src]
    j = torch.arange(have.shape[1], device=DEV)
    used = j < -(-n // page)[:, None]
    mine = used if deep else used & (j >= (n // page)[:, None])  # pages that the fork gets for itself
    ids = torch.nonzero(st["refs"] == 0)[:, 0].to(torch.int32)[: int(mine.sum())]
    _copy(st, have[mine].long(), ids.long())
    have[mine] = ids
    have[~used] = -1
    shared = have[used]
    st["refs"].index_add_(0, shared, torch.ones_like(shared))
    st["tables"][dst] = have
    st["n_kv"][dst] = n


def _grow(st, rows, add):
    page, rows = st["case"]["page"], torch.tensor(rows, device=DEV)
    n = st["n_kv"][rows]
    want = n + torch.tensor(add, device=DEV, dtype=torch.int32)
    have = st["tables"][rows]
    j = torch.arange(have.shape[1], device=DEV)
    tail = (j == (n // page)[:, None]) & (n % page != 0)[:, None] & (want > n)[:, None]  # the page that will be written on
    shared = tail & (st["refs"][have.clamp(min=0)] > 1) & (have >= 0)
    fresh = (j >= -(-n // page)[:, None]) & (j < -(-want // page)[:, None])
    mine = shared | fresh
    ids = torch.nonzero(st["refs"] == 0)[:, 0].to(torch.int32)[: int(mine.sum())]
    old = have[shared]
    have[mine] = ids
    _copy(st, old.long(), have[shared].long())
    st["refs"].index_add_(0, old, torch.full_like(old, -1))
    st["refs"][ids.long()] = 1
    st["tables"][rows] = have
    st["n_kv"][rows] = want


def _compact(st):
    live = st["refs"] > 0
    n = int(live.sum())
    holes = torch.nonzero(~live[:n])[:, 0]
    tail = torch.nonzero(live[n:])[:, 0] + n
    _copy(st, tail, holes)
    to = torch.arange(len(live), device=DEV, dtype=torch.int32)
    to[tail] = holes.to(torch.int32)
    st["tables_out"].copy_(torch.where(st["tables"] >= 0, to[st["tables"].clamp(min=0)], -1))
    st["refs_out"].copy_(st["refs"])
    st["refs_out"][holes] = st["refs"][tail]
    st["refs_out"][n:] = 0
    st["n_live"].fill_(n)


def _score(st):
    c = st["case"]
    x = st["logits"][:, : c["vocab"]].float() * c["scale"] + 0.0
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -torch.inf, 0.0, top)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    lse = top + torch.log(total)
    given = x.gather(1, st["tokens"].long()[:, None])
    st["logprob"].copy_(torch.where(given == -torch.inf, -torch.inf, given - lse)[:, 0])
    part = torch.where(e > 0, e * (x - top), 0.0).sum(-1, keepdim=True)
    st["entropy"].copy_(torch.where(total == 0, 0.0, torch.log(total) - part / total)[:, 0])
    if c["k"]:
        bits = x.view(torch.int32).long()  # as whole numbers in the order of their values, ties to the lowest index
        key = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF)) * (1 << 31) + (c["vocab"] - 1 - torch.arange(c["vocab"], device=DEV))
        ids = c["vocab"] - 1 - torch.topk(key, c["k"], dim=-1).values % (1 << 31)
        st["top_ids"].copy_(ids)
        best = x.gather(1, ids)
        st["top_logprobs"].copy_(torch.where(best == -torch.inf, -torch.inf, best - lse))


# ---- one pass ----------------------------------------------------------------------------------

_kept_by_program = {}  # the library's context


def _context():
    from moearc_b200 import Context
    if "ctx" not in _kept_by_program:
        _kept_by_program["ctx"] = Context()
    return _kept_by_program["ctx"]


def _buffer(ctx, t):
    from moearc_b200 import DeviceBuffer
    return None if t is None else DeviceBuffer(ctx, t.data_ptr(), t.numel() * t.element_size(), owned=False)


def _cache(st):
    """The cache's handle, which a program makes once and keeps beside its tensors."""
    if "cache" not in st:
        from moearc_b200.kvcache import KvCache
        c, ctx = st["case"], _context()
        st["cache"] = KvCache(ctx, n_layer=st["k"].shape[0], n_pages=st["k"].shape[1], page_tokens=c["page"], n_kv_heads=c["kv_heads"],
                              head_dim=c["dim"], kv_type=GGUF[c["kv"]], max_seq=st["tables"].shape[0], max_pages=st["tables"].shape[1],
                              n_heads=c.get("heads", 0), k_pages=[_buffer(ctx, t) for t in st["k"]], v_pages=[_buffer(ctx, t) for t in st["v"]],
                              tables=_buffer(ctx, st["tables"]), n_kv=_buffer(ctx, st["n_kv"]), refs=_buffer(ctx, st["refs"]))
        st["buffers"] = {k: _buffer(ctx, t) for k, t in st.items() if isinstance(t, torch.Tensor)}
    return st["cache"], st["buffers"]


def run(state):
    st = state
    c, op = st["case"], st["case"]["op"]
    if op == "attend":
        if own:
            cache, b = _cache(st)
            H, G, D = c["heads"], c["kv_heads"], c["dim"]
            row, size = (H + 2 * G) * D, 4
            end = c["rows"] * row * size
            new = (b["qkv"].view(H * D * size, end - H * D * size), b["qkv"].view((H + G) * D * size, end - (H + G) * D * size)) if c["append"] else (None, None)
            cache.attn_decode(0, b["out"], b["qkv"], c["rows"], H, 1.0 / D ** 0.5, q_stride=row, k_new=new[0], v_new=new[1], new_stride=row,
                              kv_begin=b.get("begin"), sinks=b.get("sinks"))
            return {"out": st["out"], "k": st["k"], "v": st["v"]}
        return _attend(st)
    if op == "score":
        if own:
            ctx = _context()
            if "buffers" not in st:
                st["buffers"] = {k: _buffer(ctx, t) for k, t in st.items() if isinstance(t, torch.Tensor)}
            b = st["buffers"]
            ctx.token_logprobs(b["logits"], GGUF[c["type"]], c["rows"], c["vocab"], row_stride=c["stride"], scale=c["scale"],
                               tokens=b["tokens"], logprob=b["logprob"], entropy=b["entropy"], k=c["k"],
                               top_ids=b["top_ids"] if c["k"] else None, top_logprobs=b["top_logprobs"] if c["k"] else None)
        else:
            _score(st)
        got = {"logprob": st["logprob"], "entropy": st["entropy"]}
        return {**got, "top_ids": st["top_ids"], "top_logprobs": st["top_logprobs"]} if c["k"] else got
    if op == "refork":
        if own:
            cache, _ = _cache(st)
            cache.free(st["dst"])
            cache.fork(st["src"], st["dst"], deep=c["deep"])
        else:
            _free(st, st["dst"], [0] * len(st["dst"]))
            _fork(st, st["src"], st["dst"], c["deep"])
    elif op == "rollback":
        if own:
            cache, _ = _cache(st)
            cache.free(st["rows"], st["keep"])
            cache.grow(st["rows"], st["add"])
        else:
            _free(st, st["rows"], st["keep"])
            _grow(st, st["rows"], st["add"])
    else:
        if own:
            cache, b = _cache(st)
            cache.compact(tables_out=b["tables_out"], refs_out=b["refs_out"], n_live=b["n_live"])
        else:
            _compact(st)
        return {"tables": st["tables_out"], "refs": st["refs_out"], "n_live": st["n_live"], "k": st["k"], "v": st["v"]}
    return {"tables": st["tables"], "refs": st["refs"], "n_kv": st["n_kv"], "k": st["k"], "v": st["v"]}


# ---- from the definitions, in 64 bits ----------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "score":
        return _exact_score(case, st)
    if case["op"] == "attend":
        return _exact_attend(case, st)
    moves = _exact_moves(case, st)
    if case["op"] == "compact":
        got = {"tables": None, "refs": None, "n_live": None}
    else:
        got = {"tables": None, "refs": None, "n_kv": None}
    for name in ("k", "v"):
        was, now = st[name], st[name].double()
        if moves:
            src, dst = (torch.tensor(m, device=DEV) for m in zip(*moves))
            for layer in range(was.shape[0]):
                now[layer][dst] = was[layer][src].double()
        got[name] = now
    return got


def _exact_attend(case, st):
    H, G, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    tables, n_kv = st["tables"].tolist(), st["n_kv"].tolist()
    begin = st["begin"].tolist() if st["begin"] is not None else [0] * len(n_kv)
    out = torch.zeros(case["rows"], H, D, dtype=torch.float64, device=DEV)
    for s, n in enumerate(n_kv):
        if n == 0:
            continue
        row = st["qkv"][s]
        if case["append"]:
            st["k"][0, tables[s][(n - 1) // page], (n - 1) % page] = row[H * D:(H + G) * D].view(G, D).to(st["k"].dtype)
            st["v"][0, tables[s][(n - 1) // page], (n - 1) % page] = row[(H + G) * D:].view(G, D).to(st["v"].dtype)
        pages = torch.tensor(tables[s][: -(-n // page)], device=DEV)
        ks, vs = (st[x][0][pages].reshape(-1, G, D)[begin[s]:n].double() for x in ("k", "v"))
        for h in range(H):
            x = ks[:, h // (H // G)] @ row[h * D:(h + 1) * D].double() / D ** 0.5
            if case["sinks"]:
                p = torch.softmax(torch.cat([x, st["sinks"][h:h + 1].double()]), 0)[:-1]
            else:
                p = torch.softmax(x, 0)
            out[s, h] = p @ vs[:, h // (H // G)]
    return {"out": out, "k": st["k"].double(), "v": st["v"].double()}


def _exact_moves(case, st):
    """The page copies of one pass, walked row by row on the host."""
    page = case["page"]
    tables, n_kv, refs = st["tables"].tolist(), st["n_kv"].tolist(), st["refs"].tolist()
    moves = []
    if case["op"] == "compact":
        n = sum(r > 0 for r in refs)
        holes = [p for p in range(n) if not refs[p]]
        return list(zip([p for p in range(n, len(refs)) if refs[p]], holes))

    def release(s, keep):
        keep = min(keep, n_kv[s])
        for j in range(-(-keep // page), -(-n_kv[s] // page)):
            refs[tables[s][j]] -= 1
            tables[s][j] = -1
        n_kv[s] = keep

    if case["op"] == "refork":
        for s in st["dst"]:
            release(s, 0)
        free = (p for p in range(len(refs)) if not refs[p])
        for a in st["src"]:
            for j in range(-(-n_kv[a] // page)):
                if case["deep"] or (j + 1) * page > n_kv[a]:
                    moves.append((tables[a][j], next(free)))
        return moves
    for s, keep in zip(st["rows"], st["keep"]):
        release(s, keep)
    free = (p for p in range(len(refs)) if not refs[p])
    for s, add in zip(st["rows"], st["add"]):
        n = n_kv[s]
        if n % page and add and refs[tables[s][n // page]] > 1:
            moves.append((tables[s][n // page], next(free)))
        for _ in range(-(-n // page), -(-(n + add) // page)):
            next(free)
    return moves


def _exact_score(case, st):
    n, k = case["rows"], case["k"]
    logprob, entropy = (torch.empty(n, dtype=torch.float64, device=DEV) for _ in range(2))
    best = torch.empty(n, k, dtype=torch.float64, device=DEV)
    for r in range(n):
        x = st["logits"][r, : case["vocab"]].double() * float(np.float32(case["scale"]))
        lp = torch.log_softmax(x, 0)
        logprob[r] = lp[int(st["tokens"][r])]
        entropy[r] = -torch.special.xlogy(lp.exp(), lp.exp()).sum()
        if k:
            best[r] = torch.topk(lp, k).values
    got = {"logprob": logprob, "entropy": entropy}
    return {**got, "top_ids": None, "top_logprobs": best} if k else got
