"""Workloads of the operators that serve sequences longer than their cache: attention with a
sliding window and sinks, attention that adds up the weight which each cached entry receives, the
choice of the entries that stay, and their move into the kept part.

`prepare` makes what a step of the engine has in hand (queries, pages, page tables, lengths),
`run` is one pass: in plain torch, or with `own` through `wpc_engine_b200.ops`.  `exact` restates
the definitions in 64 bits, one sequence and head at a time.
"""
import math

import torch

own = False

PAGE = 64
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
# query heads, key/value heads, head size: the decoder shapes of the benchmark and of the tests
SHAPES = {"7b": (28, 4, 128), "32b": (40, 8, 128), "0.5b": (14, 2, 64), "tiny": (4, 2, 16), "tiny48": (4, 2, 48)}


def listed():
    return [
        # a chat that has run far past its window: one token, latency is what counts
        dict(name="sinks decode b1", op="sinks", shape="7b", dtype="bf16", seqs=1, new=1, ctx=24577, ragged=False,
             window=4096, sinks=4),
        # a full serving batch, every sequence at another length, some shorter than the window
        dict(name="sinks decode b64 ragged", op="sinks", shape="7b", dtype="bf16", seqs=64, new=1, ctx=8000, ragged=True,
             window=2048, sinks=70),
        # a chunk of a long prompt behind 6 Ki earlier positions
        dict(name="sinks prefill 2048 of 8Ki", op="sinks", shape="7b", dtype="bf16", seqs=1, new=2048, ctx=8192,
             ragged=False, window=4096, sinks=4),
        # the 32-bit path's decode step
        dict(name="sinks decode fp32 b4", op="sinks", shape="0.5b", dtype="fp32", seqs=4, new=1, ctx=1000, ragged=True,
             window=257, sinks=5),
        # a decode step of a batch whose cache is to be cut down later
        dict(name="sums decode b8", op="sums", shape="7b", dtype="bf16", seqs=8, new=1, ctx=4001, ragged=False),
        # one long sequence
        dict(name="sums decode b1 32Ki", op="sums", shape="7b", dtype="bf16", seqs=1, new=1, ctx=32768, ragged=False),
        # a whole prompt of the benchmark
        dict(name="sums prefill 2048", op="sums", shape="7b", dtype="bf16", seqs=1, new=2048, ctx=2048, ragged=False),
        # unequal prompts of the small shape
        dict(name="sums prompts 0.5b", op="sums", shape="0.5b", dtype="bf16", seqs=16, new=1024, ctx=1024, ragged=True),
        # one layer of one sequence, cut from a page over its budget
        dict(name="select one layer", op="select", shape="7b", layers=1, seqs=1, ctx=1088, ragged=False, keep=1024,
             sinks=4, recent=256),
        # all layers of a batch after a chunk of a long prompt
        dict(name="select 28 layers b8", op="select", shape="7b", layers=28, seqs=8, ctx=4096, ragged=True, keep=2048,
             sinks=4, recent=512),
        # one sequence, all layers, from a page over its budget
        dict(name="move 28 layers b1", op="move", shape="7b", dtype="bf16", layers=28, seqs=1, ctx=1088, ragged=False,
             keep=1024, sinks=4, recent=256),
        # a batch, all layers, after a chunk of a long prompt
        dict(name="move 28 layers b8", op="move", shape="7b", dtype="bf16", layers=28, seqs=8, ctx=4096, ragged=True,
             keep=2048, sinks=4, recent=512),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sinks", "sinks", "sums", "sums", "select", "move"])
    if op in ("sinks", "sums"):
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
        shape = rng.choice(["7b", "32b", "0.5b", "tiny48"] if dtype == "bf16" else ["0.5b", "tiny", "tiny48"])
        nh = SHAPES[shape][0]
        if rng.random() < 0.5:
            new = 1
            ctx = _log_int(rng, 1, 32768 if dtype == "bf16" else 4096)
            seqs = _log_int(rng, 1, max(1, min(64, 64000 // ctx)))
        else:
            new = _log_int(rng, 2, 2048 if dtype == "bf16" else 160)
            most = 110_000_000 if dtype == "bf16" else 6_000_000
            ctx = new + rng.choice([0, _log_int(rng, 1, 6000 if dtype == "bf16" else 600)])
            ctx = min(ctx, max(new, most // (nh * new)))
            seqs = max(1, min(_log_int(rng, 1, 16), most // (nh * new * ctx)))
        case = dict(op=op, shape=shape, dtype=dtype, seqs=seqs, new=new, ctx=ctx, ragged=rng.random() < 0.6)
        if op == "sinks":
            case.update(window=_log_int(rng, 16, 4096), sinks=rng.choice([1, 4, 64, rng.randint(1, 200)]))
        return case
    keep = _log_int(rng, 64, 2048)
    case = dict(op=op, shape=rng.choice(["7b", "32b", "0.5b", "tiny"]), layers=rng.randint(1, 28), seqs=_log_int(rng, 1, 8),
                ctx=keep + _log_int(rng, 1, 2048), ragged=rng.random() < 0.6, keep=keep, sinks=rng.randint(0, 16),
                recent=_log_int(rng, 1, keep // 2 - 8))
    if op == "move":
        case["dtype"] = rng.choice(["bf16", "bf16", "fp32"]) if case["shape"] in ("0.5b", "tiny") else "bf16"
    return case


# ---- sizes of a case ------------------------------------------------------------------------------

def _lengths(case):
    """(positions of each sequence, new tokens of each): ragged ones fall evenly from the full
    length to an eighth of it, in an order that mixes long and short."""
    n, ctx, new = case["seqs"], case["ctx"], case.get("new", 1)
    if not case["ragged"]:
        return [ctx] * n, [new] * n
    order = [(i * 37 + 11) % n for i in range(n)] if n % 37 else list(range(n))
    share = [1.0 - 0.875 * k / max(n, 2) for k in order]
    lens = [max(1, int(ctx * s)) for s in share]
    return lens, [max(1, min(l, int(new * s))) for l, s in zip(lens, share)]


def _visible(case):
    """(pairs of query and visible key over all sequences, positions that any query sees)"""
    pairs = seen = 0
    lens, news = _lengths(case)
    w, s = case.get("window"), case.get("sinks", 0)
    for length, new in zip(lens, news):
        first = length - new
        if w is None:
            pairs += sum(range(first + 1, length + 1))
            seen += length
            continue
        for p in range(first, length):
            lo = max(0, p - w + 1)
            pairs += p + 1 - lo + min(s, lo)
        lo = max(0, first - w + 1)
        seen += length - lo + min(s, lo)
    return pairs, seen


def work(case):
    nh, nkv, hd = SHAPES[case["shape"]]
    lens, news = _lengths(case)
    if case["op"] in ("sinks", "sums"):
        e = 2 if case["dtype"] == "bf16" else 4
        pairs, seen = _visible(case)
        tokens = sum(news)
        b = seen * nkv * hd * 2 * e + 2 * tokens * nh * hd * e
        if case["op"] == "sums":
            b += seen * nkv * 8 + tokens * nkv * 4      # sums read and written, positions written
        return {"bytes": b, "flops": 4 * hd * nh * pairs}
    rows = case["layers"] * nkv
    keep, sinks, recent = case["keep"], case["sinks"], case["recent"]
    if case["op"] == "select":
        return {"bytes": rows * sum(8 * n + 4 * min(n, keep) for n in lens), "flops": rows * sum(lens)}
    e = 2 if case["dtype"] == "bf16" else 4
    moved = 0.0
    for n in lens:
        if n > keep:                                    # the last ones move; of the others the share that is kept
            free = n - sinks - recent
            moved += min(recent, n - keep) + max(0, n - keep - recent) * (keep - sinks - recent) / max(free, 1)
    return {"bytes": rows * (moved * 2 * (2 * hd * e + 8) + 4 * sum(min(n, keep) for n in lens)), "flops": rows * moved}


# ---- inputs ---------------------------------------------------------------------------------------

def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _table(case, gen, lens, held):
    """A page table with scrambled pages; `held(b, block)` says which blocks a sequence still has.
    One page belongs to nobody."""
    width = max((n + PAGE - 1) // PAGE for n in lens)
    want = [[held(b, i) for i in range(width)] for b in range(len(lens))]
    n_pages = sum(map(sum, want)) + 1
    perm = torch.randperm(n_pages, generator=torch.Generator().manual_seed(gen.initial_seed() % (1 << 31))).tolist()
    spare = perm.pop()
    rows = [[perm.pop() if w else -1 for w in row] for row in want]
    return _ints(rows), n_pages, spare


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    return _prepare_attention(case, gen) if case["op"] in ("sinks", "sums") else _prepare_eviction(case, gen)


def _prepare_attention(case, gen):
    nh, nkv, hd = SHAPES[case["shape"]]
    dtype = DTYPES[case["dtype"]]
    lens, news = _lengths(case)
    window, sinks = case.get("window"), case.get("sinks", 0)

    def held(b, block):
        if block * PAGE >= lens[b]:
            return False
        lo = 0 if window is None else max(0, lens[b] - news[b] - window + 1)
        return block >= lo // PAGE or block * PAGE < sinks

    table, n_pages, spare = _table(case, gen, lens, held)
    T = sum(news)
    # a direction that all queries share and the first positions' keys lie along: they draw
    # weight whatever is asked, as the first tokens of a text do
    lean = torch.randn((1, 1, hd), generator=gen, device="cuda")
    q = _normal(gen, (T, nh, hd), torch.float32) + 0.5 * lean
    k_pages = _normal(gen, (n_pages, nkv, PAGE, hd), dtype)
    v_pages = _normal(gen, (n_pages, nkv, PAGE, hd), dtype)
    k_pages[table[:, 0].long(), :, :4] = (k_pages[table[:, 0].long(), :, :4].float() + 0.7 * lean).to(dtype)
    qkv = torch.empty((T, (nh + 2 * nkv) * hd), dtype=dtype, device="cuda")        # the projection's rows
    qkv[:, : nh * hd] = q.reshape(T, nh * hd).to(dtype)
    qkv[:, nh * hd:] = 0
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    positions = [p for length, n in zip(lens, news) for p in range(length - n, length)]
    state = dict(case=case, heads=nh, kv_heads=nkv, head_dim=hd, q=qkv, k_pages=k_pages, v_pages=v_pages, table=table, spare=spare,
                 cu_seqlens=_ints(starts), ctx_lens=_ints(lens), new_lens=_ints(news),
                 seq_of_token=_ints([b for b, n in enumerate(news) for _ in range(n)]), positions=_ints(positions),
                 scale=1.0 / math.sqrt(hd), window=window, sinks=sinks, max_new=max(news), max_ctx=max(lens),
                 sums=case["op"] == "sums")
    first = [0 if window is None else max(0, length - n - window + 1) // PAGE for length, n in zip(lens, news)]
    sink_blocks = [min((sinks + PAGE - 1) // PAGE, f) for f in first]
    state["first_block"], state["sink_blocks"] = _ints(first), _ints(sink_blocks)
    state["blocks"] = max((length - 1) // PAGE - f + 1 + s for length, f, s in zip(lens, first, sink_blocks))
    if state["sums"]:
        # the sequences were cut down before: their tokens' positions lie beyond their places
        gone = 1000
        state["weight_sums"] = torch.rand((n_pages, nkv, PAGE), generator=gen, device="cuda") ** 4 * 8
        state["stored_positions"] = torch.randint(0, 1 << 20, (n_pages, nkv, PAGE), generator=gen, device="cuda",
                                                  dtype=torch.int32)
        state["token_positions"] = state["positions"] + gone
    return state


def _prepare_eviction(case, gen):
    nh, nkv, hd = SHAPES[case["shape"]]
    lens, _ = _lengths(case)
    L = case["layers"]
    table, n_pages, spare = _table(case, gen, lens, lambda b, block: block * PAGE < lens[b])
    # sums as attention leaves them: spread over decades, some entries without any weight
    shape = (L, n_pages, nkv, PAGE)
    w = torch.exp(2.5 * torch.randn(shape, generator=gen, device="cuda") - 2)
    w = torch.where(torch.rand(shape, generator=gen, device="cuda") < 0.05, torch.zeros_like(w), w)
    # entries stand in the order of an earlier cut: the kept part scrambled, the newest behind it
    C = table.shape[1] * PAGE
    lens_t = _ints(lens)
    gone = 5000
    idx = torch.arange(C, device="cuda")
    old = min(case["keep"], max(lens))
    r = torch.rand((L, len(lens), nkv, C), generator=gen, device="cuda")
    r = torch.where(idx < case["sinks"], -1.0, torch.where(idx < old, r, 2.0))     # only the kept part is scrambled
    pos = r.argsort(dim=-1, stable=True)
    pos = pos + torch.where(pos < case["sinks"], 0, gone)
    stored = torch.full(shape, 1 << 30, dtype=torch.int32, device="cuda")
    pages = torch.where(table >= 0, table, spare).long()
    stored[:, pages.reshape(-1)] = (pos.reshape(L, len(lens), nkv, -1, PAGE).permute(0, 1, 3, 2, 4)
                                    .reshape(L, -1, nkv, PAGE).to(torch.int32))
    stored[:, spare] = 1 << 30
    state = dict(case=case, weight_sums=w, stored_positions=stored, table=table, spare=spare, lens=lens_t,
                 next_positions=lens_t + gone, keep=case["keep"], sinks=case["sinks"], recent=case["recent"])
    if case["op"] == "move":
        dtype = DTYPES[case["dtype"]]
        state["k_pages"] = _normal(gen, (L, n_pages, nkv, PAGE, hd), dtype)
        state["v_pages"] = _normal(gen, (L, n_pages, nkv, PAGE, hd), dtype)
        state["kept"] = _select_plain(state)
    return state


# ---- one pass --------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        from wpc_engine_b200 import ops
        s = state
        if op == "sinks":
            return ops.attention(s["q"], s["heads"], s["kv_heads"], s["head_dim"], s["k_pages"], s["v_pages"], s["table"],
                                 s["cu_seqlens"], s["ctx_lens"], s["seq_of_token"], s["positions"], s["scale"],
                                 s["window"], s["max_new"], s["max_ctx"], sinks=s["sinks"])
        if op == "sums":
            out = ops.attention(s["q"], s["heads"], s["kv_heads"], s["head_dim"], s["k_pages"], s["v_pages"], s["table"],
                                s["cu_seqlens"], s["ctx_lens"], s["seq_of_token"], s["positions"], s["scale"], None,
                                s["max_new"], s["max_ctx"], weight_sums=s["weight_sums"],
                                stored_positions=s["stored_positions"], token_positions=s["token_positions"])
            return {"out": out, "weight_sums": s["weight_sums"], "stored_positions": s["stored_positions"]}
        if op == "select":
            return ops.select_kept(s["weight_sums"], s["stored_positions"], s["table"], s["lens"], s["next_positions"],
                                   s["keep"], s["sinks"], s["recent"])
        ops.move_kept_(s["k_pages"], s["v_pages"], s["weight_sums"], s["stored_positions"], s["table"], s["kept"])
        return {k: s[k] for k in ("k_pages", "v_pages", "weight_sums", "stored_positions")}
    if op in ("sinks", "sums"):
        return _attention_plain(state)
    return _select_plain(state) if op == "select" else _move_plain(state)


def _attention_plain(s):
    nh, nkv, hd = s["heads"], s["kv_heads"], s["head_dim"]
    B, J, Q, rep = s["table"].shape[0], s["blocks"], s["max_new"], nh // nkv
    # the blocks that a sequence's queries see: those of the sinks, then those from the window's start on
    j = torch.arange(J, device="cuda")[None, :]
    sb, first = s["sink_blocks"][:, None], s["first_block"][:, None]
    block = torch.where(j < sb, j, first + j - sb)
    block = block.clamp(max=s["table"].shape[1] - 1)
    extra = (first + j - sb >= s["table"].shape[1]) & (j >= sb)        # behind the table's end
    page = s["table"].gather(1, block.long())
    page = torch.where((page < 0) | extra, s["spare"], page).long()
    key = (block[:, :, None] * PAGE + torch.arange(PAGE, device="cuda")).reshape(B, J * PAGE)
    gone = extra[:, :, None].expand(B, J, PAGE).reshape(B, J * PAGE)
    k = s["k_pages"][page].permute(0, 2, 1, 3, 4).reshape(B, nkv, J * PAGE, hd).float()
    v = s["v_pages"][page].permute(0, 2, 1, 3, 4).reshape(B, nkv, J * PAGE, hd).float()
    seq = s["seq_of_token"].long()
    at = torch.arange(seq.numel(), device="cuda") - s["cu_seqlens"].long()[seq]
    q = torch.zeros((B, Q, nh, hd), device="cuda")
    q[seq, at] = s["q"][:, : nh * hd].float().reshape(-1, nh, hd)
    q = q.reshape(B, Q, nkv, rep, hd).permute(0, 2, 1, 3, 4).reshape(B, nkv, Q * rep, hd)
    start = (s["ctx_lens"] - s["new_lens"])[:, None]
    i = torch.arange(Q, device="cuda")[None, :]
    pos = (start + i)[:, :, None]
    seen = (key[:, None, :] <= pos) & (i < s["new_lens"][:, None])[:, :, None] & ~gone[:, None, :]
    if s["window"] is not None:
        seen &= (key[:, None, :] > pos - s["window"]) | (key[:, None, :] < s["sinks"])
    score = (q @ k.transpose(2, 3)).mul_(s["scale"]).view(B, nkv, Q, rep, J * PAGE)
    score.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total > 0, total, 1.0))
    out = (p.view(B, nkv, Q * rep, J * PAGE) @ v).view(B, nkv, Q, rep, hd).permute(0, 2, 1, 3, 4)
    out = out.reshape(B, Q, nh * hd)[seq, at].to(s["q"].dtype)
    if not s["sums"]:
        return out
    # sums over the queries and the heads of a group; this step's own entries begin with them
    w = p.sum((2, 3))
    live = ((key < s["ctx_lens"][:, None]) & ~gone)[:, None, :]
    fresh = (key >= start)[:, None, :]
    row = torch.where(live, page.repeat_interleave(PAGE, 1)[:, None, :], s["spare"])
    row = (row * nkv + torch.arange(nkv, device="cuda")[None, :, None]) * PAGE + (key % PAGE)[:, None, :]
    sums, stored = s["weight_sums"].view(-1), s["stored_positions"].view(-1)
    old = sums[row]
    sums[row] = torch.where(live, torch.where(fresh, w, old + w), old)
    token = (s["cu_seqlens"][:-1, None] + (key - start).clamp(min=0)).clamp(max=seq.numel() - 1)
    told = s["token_positions"][token.long()][:, None, :].expand(B, nkv, J * PAGE)
    stored[row] = torch.where(live & fresh, told, stored[row])
    return {"out": out, "weight_sums": s["weight_sums"], "stored_positions": s["stored_positions"]}


def _select_plain(s):
    """The stored index of the entry that belongs at each place of the kept part, int32
    [layers, sequences, kv heads, keep] (-1 behind a shorter sequence): a kept entry inside the
    kept part stays where it is, the others fill the holes in order."""
    L, _, nkv, _ = s["weight_sums"].shape
    B, keep = s["table"].shape[0], s["keep"]
    C = s["table"].shape[1] * PAGE
    page = torch.where(s["table"] < 0, s["spare"], s["table"]).long()
    w = s["weight_sums"][:, page].permute(0, 1, 3, 2, 4).reshape(L, B, nkv, C)
    pos = s["stored_positions"][:, page].permute(0, 1, 3, 2, 4).reshape(L, B, nkv, C)
    idx = torch.arange(C, device="cuda")
    n = s["lens"].long()[None, :, None, None]
    live = (idx < n).expand(L, B, nkv, C)
    safe = (pos < s["sinks"]) | (pos >= (s["next_positions"] - s["recent"])[None, :, None, None])
    rank = torch.where(live, torch.where(safe, 2, 1), 0)
    w = torch.where(safe, 0.0, torch.nan_to_num(w, nan=-math.inf, posinf=math.inf, neginf=-math.inf))
    # greatest first, ties by the lower index: by the sum, then by class, both stable
    order = w.argsort(dim=-1, descending=True, stable=True)
    order = order.gather(-1, rank.gather(-1, order).argsort(dim=-1, descending=True, stable=True))
    place = torch.empty_like(order).scatter_(-1, order, idx.expand_as(order))
    kept = (place < keep) & live
    inside = idx < keep
    hole = inside & live & ~kept
    mover = kept & ~inside
    at = torch.where(mover, mover.cumsum(-1) - 1, C)                    # the k-th mover's index, by k
    movers = torch.full((L, B, nkv, C + 1), -1, dtype=torch.int64, device="cuda").scatter_(-1, at, idx.expand_as(at))
    filled = movers.gather(-1, torch.where(hole, hole.cumsum(-1) - 1, C))
    out = torch.where(kept, idx, torch.where(hole, filled, -1))[..., : min(keep, C)].to(torch.int32)
    if keep > C:
        out = torch.cat([out, torch.full((L, B, nkv, keep - C), -1, dtype=torch.int32, device="cuda")], -1)
    return out


def _move_plain(s):
    L, _, nkv, _ = s["weight_sums"].shape
    B, keep = s["table"].shape[0], s["keep"]
    src = s["kept"].long()
    dst = torch.arange(keep, device="cuda").expand_as(src)
    none = src < 0

    def row(i):       # the row of entry i of its sequence and head, over all layers' pages
        block = (i.clamp(min=0) // PAGE).clamp(max=s["table"].shape[1] - 1)
        b = torch.arange(B, device="cuda")[None, :, None, None].expand_as(i)
        page = torch.where(none, s["spare"], s["table"].long()[b, block])
        layer = torch.arange(L, device="cuda")[:, None, None, None]
        head = torch.arange(nkv, device="cuda")[None, None, :, None]
        at = ((layer * s["weight_sums"].shape[1] + page) * nkv + head) * PAGE
        return (at + torch.where(none, 0, i % PAGE)).reshape(-1)

    a, b = row(src), row(dst)
    for name in ("k_pages", "v_pages", "weight_sums", "stored_positions"):
        t = s[name]
        flat = t.view(-1, t.shape[-1]) if t.dim() == 5 else t.view(-1)
        flat[b] = flat[a]
    return {k: s[k] for k in ("k_pages", "v_pages", "weight_sums", "stored_positions")}


# ---- the definitions in 64 bits -----------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "select":
        return torch.tensor(_exact_select(s), dtype=torch.int32)
    if case["op"] == "move":
        return _exact_move(s)
    nh, nkv, hd = s["heads"], s["kv_heads"], s["head_dim"]
    table, cu = s["table"].tolist(), s["cu_seqlens"].tolist()
    lens = s["ctx_lens"].tolist()
    out = torch.zeros((cu[-1], nh, hd), dtype=torch.float64, device="cuda")
    if s["sums"]:
        sums, stored = s["weight_sums"].double(), s["stored_positions"].clone()
    for b, length in enumerate(lens):
        t0, t1 = cu[b], cu[b + 1]
        first = length - (t1 - t0)
        if s["window"] is None:
            places = list(range(length))
        else:
            lo = max(0, first - s["window"] + 1)
            places = list(range(min(s["sinks"], lo))) + list(range(lo, length))
        at = torch.tensor(places, device="cuda")
        page = torch.tensor([table[b][p // PAGE] for p in places], device="cuda")
        pos = torch.arange(first, length, device="cuda")[:, None]
        hidden = at[None, :] > pos
        if s["window"] is not None:
            hidden = hidden | ((at[None, :] <= pos - s["window"]) & (at[None, :] >= s["sinks"]))
        for g in range(nkv):
            k, v = s["k_pages"][page, g, at % PAGE].double(), s["v_pages"][page, g, at % PAGE].double()
            received = torch.zeros(len(places), dtype=torch.float64, device="cuda")
            for h in range(g * (nh // nkv), (g + 1) * (nh // nkv)):
                x = s["q"][t0:t1, h * hd:(h + 1) * hd].double() @ k.t() * s["scale"]
                p = torch.softmax(x.masked_fill(hidden, -math.inf), dim=1)
                out[t0:t1, h] = p @ v
                received += p.sum(0)
            if s["sums"]:
                old = sums[page, g, at % PAGE]
                sums[page, g, at % PAGE] = torch.where(at >= first, received, old + received)
                stored[page[first:], g, at[first:] % PAGE] = s["token_positions"][t0:t1]
    out = out.reshape(cu[-1], nh * hd)
    return {"out": out, "weight_sums": sums, "stored_positions": stored} if s["sums"] else out


def _exact_select(s):
    sums, stored, table = s["weight_sums"].double().tolist(), s["stored_positions"].tolist(), s["table"].tolist()
    after, keep = s["next_positions"].tolist(), s["keep"]
    whole = []
    for layer in range(len(sums)):
        for b, n in enumerate(s["lens"].tolist()):
            for g in range(len(sums[layer][0])):
                w = [sums[layer][table[b][i // PAGE]][g][i % PAGE] for i in range(n)]
                p = [stored[layer][table[b][i // PAGE]][g][i % PAGE] for i in range(n)]
                safe = [x < s["sinks"] or x >= after[b] - s["recent"] for x in p]
                best = sorted(range(n), key=lambda i: (not safe[i], 0.0 if safe[i] else -w[i], i))[:keep]
                row = [i if i < n else -1 for i in range(keep)]
                chosen = set(best)
                movers = iter(sorted(i for i in best if i >= keep))
                for i in range(min(n, keep)):
                    if i not in chosen:
                        row[i] = next(movers)
                whole.append(row)
    return torch.tensor(whole).reshape(len(sums), len(after), -1, keep).tolist()


def _exact_move(s):
    names = ("k_pages", "v_pages", "weight_sums", "stored_positions")
    new = {k: s[k].clone() for k in names}
    table, kept = s["table"].tolist(), s["kept"].cpu()
    for layer in range(kept.shape[0]):
        for b in range(kept.shape[1]):
            pages = torch.tensor(table[b], device="cuda")
            for g in range(kept.shape[2]):
                src = kept[layer, b, g].long()
                dst = torch.nonzero((src >= 0) & (src != torch.arange(src.numel()))).reshape(-1)
                src, dst = src[dst].cuda(), dst.cuda()
                for k in names:
                    new[k][layer, pages[dst // PAGE], g, dst % PAGE] = s[k][layer, pages[src // PAGE], g, src % PAGE]
    return new
