"""The paged-cache operators measured: planning block tables from request lengths, appending rows with their key bounds,
selecting blocks by a bound of q.k, and attending the selected blocks.

`own` false runs plain torch forms, `own` true the library's entry points (goinfer_b200.paged). A pool holds fp16
[block][kv head][row in block][head dim], block 0 is the null block, and a cache's key bounds are [block][kv head][min, max][head dim].
"""
import functools
import math
from types import SimpleNamespace

import torch

own = False

# (query heads, kv heads, head dim) of the decoder shapes that the benchmark and the tests run, and layouts between them
LAYOUTS = ((32, 8, 128), (64, 8, 128), (32, 4, 64), (8, 8, 64), (6, 2, 128), (5, 1, 64), (28, 4, 128), (14, 2, 64))


def _plan(name, seqs, keep_lo, keep_hi, new_lo, new_hi, br):
    return {"name": name, "op": "plan", "seqs": seqs, "keep_lo": keep_lo, "keep_hi": keep_hi, "new_lo": new_lo, "new_hi": new_hi, "br": br}


def _append(name, seqs, len_lo, len_hi, new, layout, br, idle=0):
    return {"name": name, "op": "append", "seqs": seqs, "len_lo": len_lo, "len_hi": len_hi, "new": new, "kv": layout[1], "hd": layout[2], "br": br,
            "idle": idle}


def _select(name, seqs, len_lo, len_hi, layout, br, n_select, idle=0):
    return {"name": name, "op": "select", "seqs": seqs, "len_lo": len_lo, "len_hi": len_hi, "heads": layout[0], "kv": layout[1], "hd": layout[2],
            "br": br, "n_select": n_select, "idle": idle}


def _attend(name, seqs, len_lo, len_hi, layout, br, n_select, softcap=0.0, idle=0):
    return dict(_select(name, seqs, len_lo, len_hi, layout, br, n_select, idle), op="attend", softcap=softcap)


def listed():
    return [
        # a decode step of 64 sequences: drafts of up to four tokens, the rejected ones given back before the next come
        _plan("plan-decode", 64, 128, 8192, 1, 4, 16),
        # a full house turning over: prompt chunks of up to 64 tokens for 2000 sequences that keep a shared-length prefix
        _plan("plan-prompts", 2000, 0, 4096, 0, 64, 16),
        # one decode token for each of 64 sequences
        _append("append-decode", 64, 128, 8192, 1, LAYOUTS[0], 16),
        # prompt chunks of ragged place: they start and end inside blocks, and eight rows of the batch are idle
        _append("append-chunks", 7, 0, 2000, 301, LAYOUTS[2], 32, idle=8),
        # four prompts of 8192 tokens stored at once
        _append("append-prompts", 4, 0, 0, 8192, LAYOUTS[0], 64),
        # one user's next token, 8192 keys behind it
        _select("select-one", 1, 8192, 8192, LAYOUTS[0], 16, 64),
        # the benchmark's decode batch: 256 sequences of 128 to 8192 keys
        _select("select-batch", 256, 128, 8192, LAYOUTS[0], 16, 64),
        # few users with very long contexts, eight heads a group, some rows idle
        _select("select-long", 7, 60000, 131072, LAYOUTS[1], 16, 256, idle=1),
        # one user's next token over 64 selected blocks
        _attend("attend-one", 1, 8192, 8192, LAYOUTS[0], 16, 64),
        # small heads, soft-capped scores, contexts down to one token, idle rows in the batch
        _attend("attend-ragged", 45, 1, 2000, LAYOUTS[2], 32, 33, softcap=30.0, idle=3),
        # very long contexts, 256 blocks of 64 keys each
        _attend("attend-long", 4, 60000, 131072, LAYOUTS[0], 64, 256),
        # the benchmark's decode batch over 128 blocks of 16 keys a sequence
        _attend("attend-batch", 256, 2048, 8192, LAYOUTS[0], 16, 128),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("plan", "append", "select", "attend"))
    br = rng.choice((16, 16, 32, 48, 64))
    layout = rng.choice(LAYOUTS)
    idle = rng.choice((0, 0, 1, 5))
    if op == "plan":
        seqs, keep = _log(rng, 1, 2500), _log(rng, 16, 8192)
        case = _plan("", seqs, rng.randrange(keep), keep, 0, _log(rng, 1, max(1, min(4096, 65536 // seqs))), br)
    elif op == "append":
        seqs, hi = _log(rng, 1, 300), _log(rng, 16, 4096)
        case = _append("", seqs, rng.randrange(hi), hi, _log(rng, 1, max(1, 16384 // seqs)), layout, br, idle)
    else:
        # keys of all sequences together: at most a million (4 GB of pools at 8 heads of 128)
        seqs = _log(rng, 1, 256)
        hi = _log(rng, 8 * br, min(131072, 1000000 // seqs))
        lo = rng.randrange(1, hi + 1)
        n_select = _log(rng, 4, min(256, hi // br - 1))  # the longest sequences have more blocks than are selected
        if op == "select":
            case = _select("", seqs, lo, hi, layout, br, n_select, idle)
        else:
            n_select = min(n_select, max(4, 500000 // (seqs * br)))
            case = _attend("", seqs, lo, hi, layout, br, n_select, rng.choice((0.0, 0.0, 50.0)), idle)
    del case["name"]
    return case


# ---- inputs ----------------------------------------------------------------------------------------------------------


def _spread(lo, hi, n):
    """n lengths evenly over [lo, hi]."""
    return torch.linspace(lo, hi, n, dtype=torch.float64).round().to(torch.int32) if n > 1 else torch.tensor([hi], dtype=torch.int32)


def _shuffled(x, gen):
    return x.cuda()[torch.randperm(x.numel(), generator=gen, device="cuda")].contiguous()


def _tables(lens, br, spare, gen, width=0):
    """A table whose sequences hold `lens` rows in blocks of a shuffled pool, and what is left on the free stack."""
    n = lens.numel()
    blocks = (lens + br - 1) // br
    used, width = int(blocks.sum()), max(1, width, int(blocks.max()))
    n_blocks = 1 + used + spare
    ids = (torch.randperm(n_blocks - 1, generator=gen, device="cuda") + 1).to(torch.int32)
    p = torch.arange(width, device="cuda")
    at = (torch.cumsum(blocks, 0) - blocks)[:, None] + p
    table = torch.where(p < blocks[:, None], ids[at.clamp_max(n_blocks - 2)], torch.zeros((), dtype=torch.int32, device="cuda"))
    stack = torch.zeros(n_blocks, dtype=torch.int32, device="cuda")
    stack[:spare] = ids[used:]
    assert n == table.shape[0]
    return SimpleNamespace(table=table.contiguous(), blocks=blocks.to(torch.int32).contiguous(), stack=stack,
                           count=torch.tensor([spare], dtype=torch.int32, device="cuda"), n_blocks=n_blocks)


def _rows(n, n_seqs):
    i32 = functools.partial(torch.full, dtype=torch.int32, device="cuda")
    return SimpleNamespace(row0=i32((n_seqs + 1,), 0), slot=i32((n,), -1), pos=i32((n,), -1), map=i32((n,), -1), status=i32((4,), 0))


def _pool(n_blocks, case, gen):
    return torch.empty(n_blocks, case["kv"], case["br"], case["hd"], dtype=torch.float16, device="cuda").normal_(generator=gen)


def prepare(case, seed):
    gen = torch.Generator("cuda")
    gen.manual_seed(seed)
    br = case["br"]
    s = SimpleNamespace(case=case, br=br)
    if case["op"] == "plan":
        n = case["seqs"]
        s.keep = _shuffled(_spread(case["keep_lo"], case["keep_hi"], n), gen)
        s.new = _shuffled(_spread(case["new_lo"], case["new_hi"], n), gen)
        s.none = torch.zeros_like(s.new)
        spare = int(((s.new + br - 1) // br).sum()) + 7
        s.c = _tables(s.keep, br, spare, gen, (case["keep_hi"] + case["new_hi"] + br - 1) // br)
        s.rows = _rows(int(s.new.sum()) + 5, n)
        return s
    n = case["seqs"]
    lens = _shuffled(_spread(case["len_lo"], case["len_hi"], n), gen)
    total = n * case.get("new", 1)
    s.rows = _rows(total + case["idle"], n)
    r = torch.arange(total, device="cuda", dtype=torch.int32)
    if case["op"] == "append":
        s.c = _tables(lens + case["new"], br, 3, gen)
        s.rows.slot[:total] = r // case["new"]
        s.rows.pos[:total] = lens[s.rows.slot[:total].long()] + r % case["new"]
        page = s.c.table[s.rows.slot[:total].long(), (s.rows.pos[:total] // br).long()]
        s.rows.map[:total] = page * br + s.rows.pos[:total] % br
        s.k_pool, s.v_pool = _pool(s.c.n_blocks, case, gen), _pool(s.c.n_blocks, case, gen)
        s.bounds = torch.stack((s.k_pool.amin(2), s.k_pool.amax(2)), 2).contiguous()
        # k and v lie side by side in the projection's output, as the step leaves them
        kv = torch.empty(total + case["idle"], 2, case["kv"] * case["hd"], device="cuda").normal_(generator=gen)
        s.k, s.v = kv[:, 0], kv[:, 1]
        return s
    s.c = _tables(lens, br, 3, gen)
    s.rows.slot[:total] = r
    s.rows.pos[:total] = lens - 1
    s.q = torch.empty(total + case["idle"], case["heads"] * case["hd"], device="cuda").normal_(generator=gen)
    s.sel = torch.full((total + case["idle"], case["kv"], case["n_select"]), -1, dtype=torch.int32, device="cuda")
    if case["op"] == "select":
        # a block's keys scatter around a centre that drifts from block to block
        shape = (s.c.n_blocks, case["kv"], case["hd"])
        centre = torch.empty(shape, device="cuda").normal_(generator=gen)
        reach = torch.empty(shape, device="cuda").normal_(generator=gen).abs() + 0.5
        s.bounds = torch.stack((centre - reach, centre + reach), 2).half().contiguous()
        return s
    s.k_pool, s.v_pool = _pool(s.c.n_blocks, case, gen), _pool(s.c.n_blocks, case, gen)
    # a list of blocks for each row and kv head: the last block and others at random, ascending, -1 behind them
    have = ((lens + br - 1) // br)[:, None, None]
    p = torch.arange(s.c.table.shape[1], device="cuda", dtype=torch.int32)
    luck = torch.rand(n, case["kv"], p.numel(), generator=gen, device="cuda")
    luck = torch.where(p == have - 1, 2.0, torch.where(p < have, luck, -1.0))
    most = min(case["n_select"], p.numel())
    best, at = torch.topk(luck, most, dim=-1)
    at = torch.where(best >= 0, at, 1 << 30).sort(-1).values
    s.sel[:total, :, :most] = torch.where(at < 1 << 30, at, -1).to(torch.int32)
    s.out = torch.zeros(total + case["idle"], case["heads"] * case["hd"], device="cuda")
    return s


# ---- plain forms -----------------------------------------------------------------------------------------------------


def _plain_plan(c, kv_len, n_new, rows, br):
    table, cur, count = c.table, c.blocks, c.count
    n, width = table.shape
    n_rows = rows.slot.numel()
    want = (kv_len + n_new + br - 1) // br
    grow, shrink = (want - cur).clamp_min(0), (cur - want).clamp_min(0)
    total, given, taken = n_new.sum(), shrink.sum(), grow.sum()
    bad = (kv_len < 0) | (n_new < 0) | (want > width) | (kv_len > cur * br)
    any_bad = bad.any() | (total > n_rows)
    free = count[0].clone()
    missing = taken - free - given
    full = ~any_bad & (missing > 0)
    ok = ~(any_bad | full)
    p = torch.arange(width, device="cuda")
    # blocks given back: pushed with the last sequence's last block first
    back = (p >= want[:, None]) & (p < cur[:, None]) & ok
    place = free + (given - torch.cumsum(shrink, 0))[:, None] + cur[:, None] - 1 - p
    stack = torch.cat((c.stack, c.stack.new_zeros(1)))
    stack.scatter_(0, torch.where(back, place, stack.numel() - 1).reshape(-1), table.reshape(-1))
    c.stack.copy_(stack[:-1])
    table.masked_fill_(back, 0)
    # blocks taken: popped for the first sequence's first block first
    take = (p >= cur[:, None]) & (p < want[:, None]) & ok
    place = free + given - 1 - ((torch.cumsum(grow, 0) - grow)[:, None] + p - cur[:, None])
    table.copy_(torch.where(take, c.stack[place.clamp(0, c.stack.numel() - 1)], table))
    cur.copy_(torch.where(ok, want, cur))
    count.copy_(torch.where(ok, free + given - taken, free))
    r = torch.arange(n_rows, device="cuda")
    ends = torch.cumsum(n_new, 0)
    live = ok & (r < total)
    slot = torch.searchsorted(ends, r, right=True).clamp_max(n - 1)
    pos = kv_len[slot] + r - (ends - n_new)[slot]
    page = table[slot, (pos // br).clamp(0, width - 1)]
    rows.slot.copy_(torch.where(live, slot, -1))
    rows.pos.copy_(torch.where(live, pos, -1))
    rows.map.copy_(torch.where(live, page * br + pos % br, -1))
    rows.row0.zero_()
    rows.row0[1:] = torch.where(ok, ends, 0)
    first_bad = torch.where(bad.any(), bad.to(torch.int32).argmax(), n)
    rows.status.copy_(torch.stack((torch.where(any_bad, 3, torch.where(full, 2, 0)), torch.where(ok, total, 0), count[0],
                                   torch.where(any_bad, first_bad, torch.where(full, missing, 0)))))


def _plain_append(s):
    case, br, rows = s.case, s.br, s.rows
    live = torch.nonzero(rows.map >= 0)[:, 0]
    at = rows.map[live].long()
    page, row = at // br, at % br
    s.k_pool[page, :, row] = s.k[live].reshape(-1, case["kv"], case["hd"]).half()
    s.v_pool[page, :, row] = s.v[live].reshape(-1, case["kv"], case["hd"]).half()
    # the last row written in each touched block: the blocks' bounds are taken over the rows up to it
    end = torch.nonzero((torch.nn.functional.pad(at[1:], (0, 1), value=-1) != at + 1) | (row == br - 1))[:, 0]
    page, last = page[end], row[end]
    keys = s.k_pool[page]
    inside = (torch.arange(br, device="cuda") <= last[:, None])[:, None, :, None]
    low = torch.where(inside, keys, math.inf).amin(2)
    high = torch.where(inside, keys, -math.inf).amax(2)
    s.bounds[page] = torch.stack((low, high), 2)


def _plain_select(s, n_first=1, n_recent=1):
    case, br, rows = s.case, s.br, s.rows
    kv, hd, most = case["kv"], case["hd"], case["n_select"]
    live = (rows.slot >= 0)[:, None, None]
    page = s.c.table[rows.slot.clamp_min(0).long()].long()  # [row, block]
    q = s.q.double().reshape(-1, kv, 1, case["heads"] // kv, hd)
    both = s.bounds[page].transpose(1, 2).double()  # [row, kv head, block, 2, dim]
    bound = torch.where(q > 0, both[..., 1:2, :], both[..., 0:1, :])  # [row, kv head, block, head, dim]
    score = (q * bound).sum(-1).amax(-1)
    top = torch.finfo(torch.float64).max
    score = torch.nan_to_num(score, nan=top, posinf=top, neginf=-top)
    score = torch.where((page <= 0)[:, None], -top, score)
    have = (rows.pos // br + 1)[:, None, None]
    b = torch.arange(page.shape[1], device="cuda")
    score = torch.where((b < n_first) | (b >= have - n_recent), math.inf, score)
    score = torch.where(b < have, score, -math.inf)
    best, at = torch.sort(score, dim=-1, descending=True, stable=True)
    at = torch.where(best > -math.inf, at, 1 << 30)[..., :most].sort(-1).values
    found = torch.where(at < 1 << 30, at, -1).to(torch.int32)
    n = found.shape[-1]
    s.sel.copy_(torch.where(live, torch.nn.functional.pad(found, (0, most - n), value=-1), s.sel))


def _plain_attend(s):
    case, br, rows = s.case, s.br, s.rows
    kv, hd = case["kv"], case["hd"]
    group = case["heads"] // kv
    live = rows.slot >= 0
    page = s.c.table[rows.slot.clamp_min(0).long()[:, None, None], s.sel.clamp_min(0).long()].long()  # [row, kv head, entry]
    head = torch.arange(kv, device="cuda")[None, :, None]
    key = s.sel[..., None] * br + torch.arange(br, device="cuda")
    seen = (s.sel >= 0)[..., None] & (key <= rows.pos[:, None, None, None])
    seen = seen.reshape(seen.shape[0], kv, 1, -1)
    k = s.k_pool[page, head].float().reshape(page.shape[0], kv, -1, hd)
    score = torch.matmul(s.q.reshape(-1, kv, group, hd), k.transpose(-1, -2)) / math.sqrt(hd)
    del k
    if case["softcap"]:
        score = case["softcap"] * torch.tanh(score / case["softcap"])
    score = torch.where(seen, score, -math.inf)
    most = score.amax(-1, keepdim=True)
    w = torch.where(seen, torch.exp(score - torch.where(most > -math.inf, most, 0.0)), 0.0)
    total = w.sum(-1, keepdim=True)
    v = s.v_pool[page, head].float().reshape(page.shape[0], kv, -1, hd)
    o = torch.matmul(w, v) / torch.where(total > 0, total, 1.0)
    s.out.copy_(torch.where(live[:, None], o.reshape(s.out.shape), s.out))


# ---- the library's calls ---------------------------------------------------------------------------------------------


@functools.lru_cache(maxsize=None)
def _ops(stream):
    from goinfer_b200.ops import Ops
    return Ops(0, stream=stream or 1)  # torch's default stream is the legacy stream, whose handle is 1


def _cache(s):
    from goinfer_b200.paged import PagedCache, PagedRows
    ops = _ops(torch.cuda.current_stream().cuda_stream)
    s.cache = PagedCache(ops, s.c.table, s.c.blocks, s.c.stack, s.c.count, s.br, getattr(s, "k_pool", None), getattr(s, "v_pool", None),
                         getattr(s, "bounds", None))
    s.packed = PagedRows(s.rows.slot, s.rows.pos, s.rows.map, s.rows.row0, s.rows.status)
    return s.cache


def run(s):
    op = s.case["op"]
    if own:
        cache = getattr(s, "cache", None) or _cache(s)  # views over the state's buffers, which a program keeps
        if op == "plan":
            cache.plan(s.keep, s.none, s.packed)
            cache.plan(s.keep, s.new, s.packed)
        elif op == "append":
            cache.append(s.packed, s.k, s.v)
        elif op == "select":
            cache.select(s.packed, s.q, s.sel, n_first=1, n_recent=1)
        else:
            cache.attend(s.packed, s.q, s.sel, s.out, softcap=s.case["softcap"])
    elif op == "plan":
        _plain_plan(s.c, s.keep, s.none, s.rows, s.br)  # what the last step took over the kept length is given back
        _plain_plan(s.c, s.keep, s.new, s.rows, s.br)
    elif op == "append":
        _plain_append(s)
    elif op == "select":
        _plain_select(s)
    else:
        _plain_attend(s)
    if op == "plan":
        return {"row0": s.rows.row0, "slot": s.rows.slot, "pos": s.rows.pos, "map": s.rows.map, "status": s.rows.status, "table": s.c.table,
                "blocks": s.c.blocks, "stack": s.c.stack, "count": s.c.count}
    if op == "append":
        return {"k": s.k_pool, "v": s.v_pool, "bounds": s.bounds}
    return s.sel if op == "select" else s.out


# ---- what a pass cannot do without -----------------------------------------------------------------------------------


def work(case):
    n, br = case["seqs"], case["br"]
    if case["op"] == "plan":
        keep, new = _spread(case["keep_lo"], case["keep_hi"], n), _spread(case["new_lo"], case["new_hi"], n)
        rows, moved = int(new.sum()) + 5, n * (float(new.double().mean()) / br)
        assert keep.numel() == n
        # per call: lengths and block counts in, counts and offsets out, three numbers a row; a moved block: table and stack
        return {"bytes": 2 * 4 * (3 * n + 2 * n + 3 * rows) + 2 * 8 * moved, "flops": 0}
    if case["op"] == "append":
        rows, tile = n * case["new"], case["kv"] * case["hd"]
        lens = _spread(case["len_lo"], case["len_hi"], n)
        first, last = lens // br, (lens + case["new"] - 1) // br
        touched, older = int((last - first + 1).sum()), int((lens % br).sum())
        return {"bytes": rows * (tile * 12 + 4) + touched * tile * 4 + older * tile * 2, "flops": 2 * rows * tile}
    lens = _spread(case["len_lo"], case["len_hi"], n).long()
    have = (lens + br - 1) // br
    qo = n * case["heads"] * case["hd"] * 4
    listed_ = n * case["kv"] * case["n_select"] * 4
    if case["op"] == "select":
        scored = int(torch.where(have > case["n_select"], have - 2, 0).sum()) * case["kv"]
        return {"bytes": qo + listed_ + scored * case["hd"] * 4, "flops": 2 * scored * case["hd"] * case["heads"] // case["kv"]}
    full = torch.minimum(have, torch.tensor(case["n_select"]))
    keys = int((full * br - (have * br - lens)).sum()) * case["kv"]
    return {"bytes": 2 * qo + listed_ + keys * case["hd"] * 4, "flops": 4 * keys * case["hd"] * case["heads"] // case["kv"]}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------


def exact(case, seed):
    if case["op"] in ("plan", "select"):
        return None  # whole numbers
    s = prepare(case, seed)
    br, kv, hd = s.br, case["kv"], case["hd"]
    if case["op"] == "append":
        k, v, bounds = s.k_pool.double(), s.v_pool.double(), s.bounds.double()
        maps = s.rows.map.tolist()
        touched = {}
        for r, at in enumerate(maps):
            if at >= 0:
                touched[at // br] = max(touched.get(at // br, 0), at % br)
        index = torch.tensor([a for a in maps if a >= 0], device="cuda")
        rows = torch.tensor([r for r, a in enumerate(maps) if a >= 0], device="cuda")
        # a stored value is the nearest fp16 value, ties to even
        k.transpose(1, 2)[index // br, index % br] = s.k[rows].half().double().reshape(-1, kv, hd)
        v.transpose(1, 2)[index // br, index % br] = s.v[rows].half().double().reshape(-1, kv, hd)
        for page, last in touched.items():
            bounds[page, :, 0] = k[page, :, : last + 1].min(1).values
            bounds[page, :, 1] = k[page, :, : last + 1].max(1).values
        return {"k": k, "v": v, "bounds": bounds}
    out = s.out.double()
    group = case["heads"] // kv
    tables, sels = s.c.table.tolist(), s.sel.tolist()
    slots, poss = s.rows.slot.tolist(), s.rows.pos.tolist()
    for r, (slot, pos) in enumerate(zip(slots, poss)):
        if slot < 0:
            continue
        for h in range(kv):
            blocks = [b for b in sels[r][h] if b >= 0]
            pages = torch.tensor([tables[slot][b] for b in blocks], device="cuda")
            keys = torch.tensor(blocks, device="cuda")[:, None] * br + torch.arange(br, device="cuda")
            seen = keys.reshape(-1) <= pos
            k = s.k_pool[pages, h].double().reshape(-1, hd)[seen]
            v = s.v_pool[pages, h].double().reshape(-1, hd)[seen]
            q = s.q[r].double().reshape(kv, group, hd)[h]
            x = q @ k.T / math.sqrt(hd)
            if case["softcap"]:
                x = case["softcap"] * torch.tanh(x / case["softcap"])
            out[r].reshape(kv, group, hd)[h] = torch.softmax(x, -1) @ v
    return out
