"""What serving endless streams is timed on: attention over a window and a stream's first positions, the paged cache's tables
built on the GPU, and keys and values stored by slot map.

A case is one operator at one size.  `run` makes one pass through it: with `own` the calls a program makes of
`lastengine_b200.ops.kernels`, without it the same numbers from elementary torch operations in 32 bits.  The lengths of a
case's sequences are spread evenly, on a logarithmic scale, between the two that it names.

The cache is the framework's: pages of `page` positions, keys [page][kv head][position][dim], values [page][kv head][dim]
[position], a page list per sequence with -1 where a page has been given back.  A row at position p sees position j <= p
where j > p - window or j < first.
"""
from __future__ import annotations

import math
import types

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---- the cases -------------------------------------------------------------------------------------------------------
def _attention(name, type="bf16", heads=32, kv_heads=8, dim=64, vdim=64, seqs=1, padding=0, new=(1, 1), held=(0, 0),
               window=1024, first=4, page=64):
    return {"name": name, "op": "attention", "type": type, "heads": heads, "kv_heads": kv_heads, "dim": dim, "vdim": vdim,
            "seqs": seqs, "padding": padding, "new_lo": new[0], "new_hi": new[1], "held_lo": held[0], "held_hi": held[1],
            "window": window, "first": first, "page": page}


def _store(name, type="bf16", heads=32, kv_heads=8, dim=64, vdim=64, seqs=1, new=(1, 1), held=(0, 0), page=64):
    return {"name": name, "op": "store", "type": type, "heads": heads, "kv_heads": kv_heads, "dim": dim, "vdim": vdim,
            "seqs": seqs, "new_lo": new[0], "new_hi": new[1], "held_lo": held[0], "held_hi": held[1], "page": page}


def _tables(name, seqs=1, padding=0, new=(1, 1), held=(0, 0), window=1024, first=4, page=64, advance=True):
    return {"name": name, "op": "tables", "seqs": seqs, "padding": padding, "new_lo": new[0], "new_hi": new[1],
            "held_lo": held[0], "held_hi": held[1], "window": window, "first": first, "page": page, "advance": advance}


def listed():
    return [
        # one conversation's decode step: every call's fixed cost counts
        _attention("token, one stream", held=(1500, 1500)),
        # a serving batch's decode step, streams of all ages, three places of the captured step's bucket empty
        _attention("token, 64 streams", seqs=61, padding=3, held=(20, 30000), window=4096, first=64),
        # the 32-bit path's decode step, heads of an odd width and values of their own
        _attention("token, 32-bit, odd heads", type="f32", heads=15, kv_heads=5, dim=80, vdim=48, seqs=7, held=(1, 3001), window=777, first=5),
        # new prompts and further turns of old conversations in one step
        _attention("turns of 12 streams", seqs=12, new=(3, 1500), held=(0, 6000), window=1024, first=16),
        # wide heads
        _attention("turns, heads of 128", heads=16, kv_heads=4, dim=128, vdim=128, seqs=4, new=(100, 2047), held=(0, 3000), window=2048, first=4),
        # a document read in one step
        _attention("document", new=(8191, 8191), window=4096, first=128),
        # the same of a decode step's tables: one stream that goes on
        _tables("tables, one stream", held=(5000, 5000)),
        # a serving batch: most streams decode, rows and pages of all ages
        _tables("tables, 64 streams", seqs=61, padding=3, held=(1, 30000), window=4096, first=64),
        # a step that admits many prompts beside many streams: the tables only, as before a step's first layer
        _tables("tables, 1000 prompts", seqs=1000, new=(1, 900), held=(0, 20000), window=4096, first=100, advance=False),
        # a decode step's keys and values, cut from the fused projection
        _store("store, 64 tokens", seqs=64, held=(1, 30000)),
        # the 32-bit path, odd widths, ragged prompts
        _store("store, 32-bit, odd heads", type="f32", heads=6, kv_heads=3, dim=80, vdim=48, seqs=5, new=(7, 701), held=(0, 999), page=32),
        # a step of prompts
        _store("store, prompts", seqs=16, new=(64, 4000), held=(0, 2000)),
    ]


def _log_int(rng, lo, hi):
    return min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "tables", "tables", "store", "store"])
    page = rng.choice([64, 64, 64, 64, 32, 128])
    window, first = _log_int(rng, 16, 6000), rng.choice([1, 4, 4, _log_int(rng, 1, 300)])
    held = sorted((_log_int(rng, 1, 30000) - 1, _log_int(rng, 1, 30000)))
    if op == "tables":
        seqs = _log_int(rng, 1, 1000)
        new = sorted((_log_int(rng, 1, 900), _log_int(rng, 1, 900))) if rng.random() < 0.6 else [1, 1]
        held[1] = min(held[1], 20000)
        held[0] = min(held)
        c = _tables("", seqs=seqs, padding=rng.choice([0, 0, 1, 5]), new=new, held=held, window=window, first=first,
                    page=page, advance=rng.random() < 0.6)
    else:
        kv = rng.choice([1, 2, 3, 4, 8])
        group = rng.choice([1, 2, 3, 4, 5, 8, 16] if kv <= 2 else [1, 2, 3, 4])
        type = rng.choice(["bf16", "bf16", "bf16", "f32"])
        dim = rng.choice([32, 64, 64, 64, 96, 128, 128] if type == "bf16" else [32, 48, 64, 80, 128])
        turns = op == "attention" and rng.random() < 0.5
        if not turns and rng.random() < 0.15:
            dim = rng.choice([80, 192])
        vdim = rng.choice([32, 48, 64]) if rng.random() < 0.25 and not (turns and type == "bf16") else dim
        if op == "store":
            seqs = _log_int(rng, 1, 64)
            new = sorted((_log_int(rng, 1, 16000 // seqs), _log_int(rng, 1, 16000 // seqs))) if rng.random() < 0.6 else [1, 1]
            c = _store("", type=type, heads=kv * group, kv_heads=kv, dim=dim, vdim=vdim, seqs=seqs, new=new, held=held, page=page)
        elif not turns:
            c = _attention("", type=type, heads=kv * group, kv_heads=kv, dim=dim, vdim=vdim, seqs=_log_int(rng, 1, 60 if type == "bf16" else 20),
                           padding=rng.choice([0, 0, 2]), held=held, window=window, first=first, page=page)
        else:
            seqs = _log_int(rng, 1, 8)
            top = _log_int(rng, 2, 4000 // seqs if type == "bf16" else 900 // seqs)
            c = _attention("", type=type, heads=kv * group, kv_heads=kv, dim=dim, vdim=vdim, seqs=seqs, new=sorted((_log_int(rng, 1, top), top)),
                           held=sorted((rng.randrange(4000), rng.randrange(4000))), window=window, first=first, page=page)
    del c["name"]
    return c


def _spread(lo, hi, n, turn):
    """n whole numbers from lo to hi, evenly on a logarithmic scale, in an order that `turn` shifts."""
    v = [lo if n == 1 else int(round((lo + 1) * ((hi + 1) / (lo + 1)) ** (i / (n - 1)))) - 1 for i in range(n)]
    return [v[(i * 7 + turn) % n] if math.gcd(7, n) == 1 else v[(i + turn) % n] for i in range(n)]


def _lengths(case):
    """(tokens a sequence brings, positions it held before) of every sequence, padding last (one row each)."""
    n, pad = case["seqs"], case.get("padding", 0)
    return (_spread(case["new_lo"], case["new_hi"], n, 0) + [1] * pad, _spread(case["held_lo"], case["held_hi"], n, 3) + [0] * pad)


def work(case):
    new, held = _lengths(case)
    rows = sum(new)
    if case["op"] == "tables":
        P, n, pad = case["page"], case["seqs"], case.get("padding", 0)
        width = -(-max(a + b for a, b in zip(new, held)) // P)
        live = sum(-(-a // P) for a in held)
        words = 3 * rows + 6 * (n + pad) + (n + pad) * width + live       # rows, sequences, the tables and what they are made of
        if case["advance"]:
            words += 4 * n
        return {"bytes": 4 * words, "flops": 0}
    size = 2 if case["type"] == "bf16" else 4
    width = case["dim"] + case["vdim"]
    if case["op"] == "store":
        return {"bytes": 2 * rows * case["kv_heads"] * width * size + 4 * rows, "flops": 0}
    w, f = case["window"], case["first"]
    pairs = cached = 0            # pairs of a row and a position it sees, positions that any row sees
    for n, h in zip(new[:case["seqs"]], held):
        lo = max(0, h + 1 - w)
        cached += h + n - lo + min(f, lo)
        for p in range(h, h + n):
            lo = max(0, p + 1 - w)
            pairs += p + 1 - lo + min(f, lo)
    return {"bytes": size * (rows * case["heads"] * width + cached * case["kv_heads"] * width), "flops": 2 * pairs * case["heads"] * width}


# ---- what a program has in hand --------------------------------------------------------------------------------------
def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _paged(case, seed, gen, full):
    """Page lists of the case's sequences: (table of what is held before the step, the same after it, pages in all, free pages).
    `full`: nothing has been given back."""
    P = case["page"]
    new, held = _lengths(case)
    n, live = len(new), case["seqs"]
    width = -(-max(a + b for a, b in zip(new, held)) // P)
    h, t = (torch.tensor(v, device="cuda") for v in (held, [a + b for a, b in zip(new, held)]))
    j = torch.arange(width, device="cuda")
    alive = (torch.arange(n, device="cuda") < live)[:, None]
    kept = torch.ones_like(h)[:, None].bool() if full else (j * P < case["first"]) | ((j[None] + 1) * P > (h + 1 - case["window"])[:, None])
    before = alive & kept & (j * P < h[:, None])
    after = alive & kept & (j * P < t[:, None])
    n_pages = int(after.sum()) + 5
    ids = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    count = torch.cumsum(after.reshape(-1).int(), 0).reshape(after.shape).long() - 1
    table = torch.where(after, ids[count.clamp(min=0)], -1).to(torch.int32)
    return torch.where(before, table, -1).to(torch.int32), table, n_pages, ids


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    P = case["page"]
    new, held = _lengths(case)
    n, rows = len(new), sum(new)
    start = [0] * n
    for i in range(1, n):
        start[i] = start[i - 1] + new[i - 1]
    s = types.SimpleNamespace(case=case)
    if case["op"] == "tables":
        before, after, n_pages, ids = _paged(case, seed, gen, False)
        width = before.shape[1]
        S = n + 3                                    # slots of the cache, in another order than the step's sequences
        slots = torch.randperm(S, generator=gen, device="cuda")[:n].to(torch.int32)
        live = torch.arange(n, device="cuda") < case["seqs"]
        s.seq_slot = torch.where(live, slots, -1).to(torch.int32)
        s.seq_qlen = _ints(new)
        # the tables' state in one buffer, so that it can be saved and put back by one copy
        sizes = {"lens": S, "kept": S, "pages": S * width, "free": n_pages, "counts": 2}
        offs, at = {}, 0
        for k, v in sizes.items():
            offs[k] = at
            at += -(-v // 4) * 4
        s.saved = torch.zeros(at, dtype=torch.int32, device="cuda")
        s.state = torch.zeros(at, dtype=torch.int32, device="cuda")
        v = {k: s.saved[offs[k]:offs[k] + m] for k, m in sizes.items()}
        fp = -(-case["first"] // P)
        gone = (torch.tensor(held, device="cuda") + 1 - case["window"]).clamp(min=0) // P
        at_slot = slots[:case["seqs"]].long()
        v["lens"][at_slot] = _ints(held)[:case["seqs"]]
        v["kept"].fill_(fp)
        v["kept"][at_slot] = gone.clamp(min=fp)[:case["seqs"]].to(torch.int32)
        v["pages"].fill_(-1)
        v["pages"].view(S, width)[at_slot] = before[:case["seqs"]]
        used = torch.zeros(n_pages, dtype=torch.bool, device="cuda")
        used[before[before >= 0].long()] = True
        free = ids[~used[ids.long()]]
        v["free"][:free.numel()] = free
        v["counts"][0] = free.numel()
        s.state.copy_(s.saved)
        for k, m in sizes.items():
            setattr(s, k, s.state[offs[k]:offs[k] + m])
        s.pages = s.pages.view(S, width)
        empty = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")
        s.table, s.slot_map, s.row_seq, s.row_pos = empty(n, width), empty(rows), empty(rows), empty(rows)
        s.step_slot, s.step_qlen, s.pos0, s.qstart = empty(n), empty(n), empty(n), empty(n)
        return s
    dtype, nh, nkv, hd, vd = TYPES[case["type"]], case["heads"], case["kv_heads"], case["dim"], case["vdim"]
    full = case["op"] == "store"
    before, table, n_pages, _ = _paged(case, seed, gen, full)
    s.k_pool = torch.randn((n_pages, nkv, P, hd), generator=gen, device="cuda").to(dtype)
    s.v_pool = torch.randn((n_pages, nkv, vd, P), generator=gen, device="cuda").to(dtype)
    row_seq = torch.repeat_interleave(torch.arange(n, device="cuda"), torch.tensor(new, device="cuda"))
    row_pos = torch.arange(rows, device="cuda") - torch.tensor(start, device="cuda")[row_seq] + torch.tensor(held, device="cuda")[row_seq]
    if full:
        # k and v as columns of the fused projection of q, k and v
        proj = torch.randn((rows, nh * hd + nkv * (hd + vd)), generator=gen, device="cuda").to(dtype)
        s.k_in, s.v_in = proj[:, nh * hd:(nh + nkv) * hd], proj[:, (nh + nkv) * hd:]
        s.slot_map = (table[row_seq, row_pos // P].long() * P + row_pos % P).to(torch.int32)
        return s
    # normed queries; a stream's first keys draw more of every query's weight than others, as they do in trained models
    lean = torch.randn((nkv, 1, hd), generator=gen, device="cuda")
    s.q = (torch.randn((rows, nkv, nh // nkv, hd), generator=gen, device="cuda") + 0.5 * lean).reshape(rows, nh * hd).to(dtype)
    if case["first"] > 0:
        top = table[:case["seqs"], 0].long()
        s.k_pool[top, :, :min(4, case["first"], P)] += (0.5 * lean).to(dtype)
    s.table, s.out = table, torch.zeros((rows, nh * vd), dtype=dtype, device="cuda")
    live = torch.arange(n, device="cuda") < case["seqs"]
    s.batch = types.SimpleNamespace(
        n_rows=rows, n_seqs=n, max_qlen=max(new), max_kvlen=max(a + b for a, b in zip(new, held)),
        row_seq=row_seq.to(torch.int32), row_pos=row_pos.to(torch.int32),
        seq_slot=torch.where(live, torch.arange(n, device="cuda"), -1).to(torch.int32),
        seq_pos0=_ints(held), seq_qstart=_ints(start), seq_qlen=_ints(new))
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------
def _own_pass(s):
    from lastengine_b200.ops import kernels
    c = s.case
    if c["op"] == "tables":
        if c["advance"]:
            s.state.copy_(s.saved)
        kernels.stream_tables(s.table, s.slot_map, s.row_seq, s.row_pos, s.step_slot, s.step_qlen, s.pos0, s.qstart,
                              s.seq_slot, s.seq_qlen, s.lens, s.pages, s.free, s.counts, c["page"])
        if c["advance"]:
            kernels.stream_advance(s.step_slot, s.step_qlen, s.lens, s.kept, s.pages, s.free, s.counts, c["page"], c["window"], c["first"])
        return
    if c["op"] == "store":
        kernels.store_rows(s.k_pool, s.v_pool, s.k_in, s.v_in, s.slot_map)
        return
    nh, nkv, hd, vd = c["heads"], c["kv_heads"], c["dim"], c["vdim"]
    n = kernels.attention_splits(s.batch, nkv, nh // nkv, hd=hd, window=c["window"], first=c["first"],
                                 general=c["type"] == "f32" or vd != hd)
    scratch = torch.empty(s.batch.n_rows * nh * n * (max(hd, vd) + 2), dtype=torch.float32, device="cuda") if n > 1 else None
    kernels.attention(s.out, s.q, s.k_pool, s.v_pool, s.table, s.batch, nh, nkv, hd, c["page"], c["window"], hd ** -0.5,
                      n_splits=n, scratch=scratch, vd=vd, first=c["first"])


def _plain_tables(s):
    c, P = s.case, s.case["page"]
    if c["advance"]:
        s.state.copy_(s.saved)
    live = s.seq_slot >= 0
    slot = s.seq_slot.clamp(min=0).long()
    qlen = s.seq_qlen.long()
    pos0 = torch.where(live, s.lens[slot], 0).long()
    end = torch.cumsum(qlen, 0)
    qstart = end - qlen
    r = torch.arange(s.row_seq.numel(), device="cuda")
    row_seq = torch.searchsorted(end, r, right=True)
    row_pos = pos0[row_seq] + r - qstart[row_seq]
    had = (pos0 + P - 1) // P
    need = torch.where(live, (pos0 + qlen + P - 1) // P - had, 0)
    taken = torch.cumsum(need, 0) - need
    j = torch.arange(s.table.shape[1], device="cuda")[None]
    at = s.counts[0].long() - 1 - (taken - had)[:, None] - j
    fresh = s.free[at.clamp(0, s.free.numel() - 1)]
    table = torch.where(j < had[:, None], s.pages[slot, :s.table.shape[1]], torch.where(j < (had + need)[:, None], fresh, -1))
    table = torch.where(live[:, None], table, -1)
    s.table.copy_(table)
    s.slot_map.copy_(torch.where(live[row_seq], table[row_seq, row_pos // P] * P + row_pos % P, -1))
    s.row_seq.copy_(row_seq)
    s.row_pos.copy_(row_pos)
    s.step_slot.copy_(s.seq_slot)
    s.step_qlen.copy_(s.seq_qlen)
    s.pos0.copy_(pos0)
    s.qstart.copy_(qstart)
    if not c["advance"]:
        s.pages[slot[live], :table.shape[1]] = table[live]
        return
    # the sequences are longer, the pages taken leave the stack, those no later row sees go back on it
    now = pos0 + qlen
    kept = s.kept[slot].long()
    gone = (now + 1 - c["window"]).clamp(min=0) // P if c["window"] > 0 else torch.zeros_like(now)
    keep = torch.maximum(kept, gone)
    back = live[:, None] & (j >= kept[:, None]) & (j < keep[:, None])
    given = table[back]
    top = s.counts[0].long() - need.sum()
    s.free[top + torch.arange(given.numel(), device="cuda")] = given
    s.counts[0] = top + given.numel()
    s.pages[slot[live], :table.shape[1]] = torch.where(back, -1, table)[live]
    s.lens[slot[live]] = now[live].to(torch.int32)
    s.kept[slot[live]] = keep[live].to(torch.int32)


def _plain_store(s):
    P, nkv = s.case["page"], s.case["kv_heads"]
    page, off = s.slot_map.long() // P, s.slot_map.long() % P
    rows = s.slot_map.numel()
    head = torch.arange(nkv, device="cuda")[None]
    s.k_pool[page[:, None], head, off[:, None]] = s.k_in.reshape(rows, nkv, -1)
    s.v_pool[page[:, None], head, :, off[:, None]] = s.v_in.reshape(rows, nkv, -1)


def _plain_attention(s):
    c, b, P = s.case, s.batch, s.case["page"]
    nh, nkv, hd, vd = c["heads"], c["kv_heads"], c["dim"], c["vdim"]
    B, Q, T = b.n_seqs, b.max_qlen, b.max_kvlen
    t, i, head = torch.arange(T, device="cuda"), torch.arange(Q, device="cuda"), torch.arange(nkv, device="cuda")
    page = s.table.long().clamp(min=0)[:, t // P]                                         # [B, T]
    k = s.k_pool[page[:, None], head[None, :, None], (t % P)[None, None]].float()         # [B, kv head, T, dim]
    v = s.v_pool[page[:, None], head[None, :, None], :, (t % P)[None, None]].float()
    rows = (b.seq_qstart.long()[:, None] + i).clamp(max=b.n_rows - 1)
    q = s.q[rows].float().view(B, Q, nkv, nh // nkv, hd).permute(0, 2, 3, 1, 4).reshape(B, nkv, nh // nkv * Q, hd)
    x = torch.matmul(q, k.transpose(2, 3)).mul_(hd ** -0.5).view(B, nkv, nh // nkv, Q, T)
    pos = b.seq_pos0.long()[:, None] + i                                                  # [B, Q]
    lo = pos[:, :, None] - c["window"]
    sees = (t <= pos[:, :, None]) & ((t > lo) | (t < c["first"])) & (b.seq_slot >= 0)[:, None, None]
    x.masked_fill_(~sees[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True).clamp_(min=torch.finfo(torch.float32).min)             # a row that sees nothing: exp(-inf)
    x.sub_(top).exp_()
    total = x.sum(-1).unsqueeze(-1)
    o = torch.matmul(x.view(B, nkv, nh // nkv * Q, T), v).view(B, nkv, nh // nkv, Q, vd)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(B, Q, nh * vd)
    seq = b.row_seq.long()
    s.out.copy_(o[seq, b.row_pos.long() - b.seq_pos0.long()[seq]])


def run(state):
    if own:
        _own_pass(state)
    else:
        {"tables": _plain_tables, "store": _plain_store, "attention": _plain_attention}[state.case["op"]](state)
    s = state
    if s.case["op"] == "tables":
        return {k: getattr(s, k) for k in ("table", "slot_map", "row_seq", "row_pos", "step_slot", "step_qlen", "pos0", "qstart",
                                           "lens", "kept", "pages", "free", "counts")}
    return {"k": s.k_pool, "v": s.v_pool} if s.case["op"] == "store" else s.out


# ---- the definition, in 64 bits --------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "tables":
        return None
    s = prepare(case, seed)
    P, nkv, hd, vd = case["page"], case["kv_heads"], case["dim"], case["vdim"]
    new, held = _lengths(case)
    if case["op"] == "store":
        k, v = s.k_pool.double(), s.v_pool.double()
        slots = s.slot_map.tolist()
        for lo in range(0, len(slots), 1000):
            part = torch.tensor(slots[lo:lo + 1000], device="cuda")
            for h in range(nkv):
                k[part // P, h, part % P] = s.k_in[lo:lo + 1000, h * hd:(h + 1) * hd].double()
                for d in range(vd):
                    v[part // P, h, d, part % P] = s.v_in[lo:lo + 1000, h * vd + d].double()
        return {"k": k, "v": v}
    G = case["heads"] // nkv
    out = torch.zeros((sum(new), nkv, G, vd), dtype=torch.float64, device="cuda")
    table, row = s.table.tolist(), 0
    for b, (n, h) in enumerate(zip(new, held)):
        for q0 in range(h, h + n if b < case["seqs"] else h, 512):
            m = min(512, h + n - q0)
            lo = max(0, q0 + 1 - case["window"])      # what the first of these rows sees; what the last one sees ends with itself
            at = list(range(min(case["first"], lo))) + list(range(lo, q0 + m))
            pages = torch.tensor([table[b][j // P] for j in at], device="cuda")
            t = torch.tensor(at, device="cuda")
            p = torch.arange(q0, q0 + m, device="cuda")[:, None]
            hidden = (t > p) | ((t >= case["first"]) & (t + case["window"] <= p))
            for g in range(nkv):
                k = s.k_pool[pages, g, t % P].double()
                v = s.v_pool[pages, g, :, t % P].double()
                r0 = row + q0 - h
                for hh in range(G):
                    q = s.q[r0:r0 + m, (g * G + hh) * hd:(g * G + hh + 1) * hd].double()
                    w = torch.softmax((q @ k.t() / math.sqrt(hd)).masked_fill(hidden, -math.inf), -1)
                    out[r0:r0 + m, g, hh] = w @ v
        row += n
    return out.view(sum(new), -1)
