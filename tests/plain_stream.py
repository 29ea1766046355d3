"""Plain implementations beside which the stream kernels are tested: the bookkeeping as lists of whole numbers, and
attention over a window and a sequence's first positions in double precision."""
import math

import numpy as np
import torch


class PlainTables:
    """Page lists of endless streams: what csrc/stream_tables.cu does, one sequence and one page at a time."""

    def __init__(self, n_pages, n_slots, width, page, window, first, free=None):
        self.page, self.window, self.first, self.width = page, window, first, width
        self.lens = [0] * n_slots
        self.lists = [[] for _ in range(n_slots)]
        self.free = list(range(n_pages - 1, -1, -1)) if free is None else list(free)
        self.n_pages = n_pages

    def tables(self, slots, qlens, n_rows, width=None):
        """The step's tables, or the status of a step that is refused."""
        width = min(width or self.width, self.width)
        P = self.page
        if any(s < -1 or s >= len(self.lens) for s in slots) or any(n < 0 for n in qlens):
            return -3
        if any(s >= 0 and self.lens[s] + n > width * P for s, n in zip(slots, qlens)):
            return -1
        if sum(qlens) != n_rows:
            return -2
        need = [0 if s < 0 else -(-(self.lens[s] + n) // P) - len(self.lists[s]) for s, n in zip(slots, qlens)]
        if sum(need) > len(self.free):
            return sum(need) - len(self.free)
        out = {k: [] for k in ("table", "slot_map", "row_seq", "row_pos", "pos0", "qstart")}
        taken = 0
        for b, (s, n) in enumerate(zip(slots, qlens)):
            pages = [] if s < 0 else self.lists[s] + [self.free[-1 - taken - i] for i in range(need[b])]
            taken += need[b]
            pos0 = 0 if s < 0 else self.lens[s]
            out["qstart"].append(len(out["row_seq"]))
            out["pos0"].append(pos0)
            out["table"].append(pages)
            for i in range(n):
                out["row_seq"].append(b)
                out["row_pos"].append(pos0 + i)
                out["slot_map"].append(-1 if s < 0 else pages[(pos0 + i) // P] * P + (pos0 + i) % P)
        return out

    def advance(self, slots, qlens, tables):
        P, taken = self.page, 0
        for s, n, pages in zip(slots, qlens, tables["table"]):
            if s >= 0:
                taken += len(pages) - len(self.lists[s])
                self.lists[s] = list(pages)
                self.lens[s] += n
        del self.free[len(self.free) - taken:]
        for s in slots:
            if s < 0 or self.window <= 0:
                continue
            seen_from = self.lens[s] + 1 - self.window      # by the next row
            for j, p in enumerate(self.lists[s]):
                if p >= 0 and j * P >= self.first and (j + 1) * P <= seen_from:
                    self.free.append(p)
                    self.lists[s][j] = -1

    def release(self, slots):
        for s in slots:
            if s >= 0:
                self.free += [p for p in self.lists[s] if p >= 0]
                self.lists[s], self.lens[s] = [], 0


def sees(pos, t, window, first):
    """[rows, positions]: whether the row at `pos` sees position t."""
    ok = t[None] <= pos[:, None]
    if window > 0:
        ok &= (t[None] > pos[:, None] - window) | (t[None] < first)
    return ok


def attention(q, k, v, pos, window, first, scale, slopes=None, sinks=None):
    """(result, sum of weights times |values|, largest sum of |q k| scale of a row's pairs) in double precision.
    q [rows, heads, width], k and v [positions, kv heads, width]; only positions that a row sees are touched."""
    rows, nh, _ = q.shape
    G = nh // k.shape[1]
    out = torch.zeros(rows, nh, v.shape[2], dtype=torch.float64)
    mass = torch.zeros_like(out)
    size = torch.zeros(rows, nh, 1, dtype=torch.float64)
    t = torch.arange(k.shape[0])
    ok = sees(pos, t, window, first)
    seen = ok.any(0)
    kc, vc = torch.where(seen[:, None, None], k, 0.0), torch.where(seen[:, None, None], v, 0.0)
    for h in range(nh):
        s = (q[:, h] @ kc[:, h // G].T) * scale
        if slopes is not None:
            s = s - slopes[h] * (pos[:, None] - t[None])
        s = s.masked_fill(~ok, -math.inf)
        if sinks is not None:
            w = torch.softmax(torch.cat([s, torch.full((rows, 1), float(sinks[h]), dtype=torch.float64)], 1), -1)[:, :-1]
        else:
            w = torch.softmax(s, -1)
        out[:, h] = w @ vc[:, h // G]
        mass[:, h] = w @ vc[:, h // G].abs()
        size[:, h, 0] = ((q[:, h].abs() @ kc[:, h // G].abs().T) * scale).masked_fill(~ok, 0.0).amax(-1)
    return out, mass, size


def random_lists(rng, lens, page, n_extra=3):
    """A page list per sequence of `lens` positions, pages in random order; how many pages there are."""
    need = [-(-n // page) for n in lens]
    ids = rng.permutation(sum(need) + n_extra)
    out, at = [], 0
    for n in need:
        out.append([int(p) for p in ids[at:at + n]])
        at += n
    return out, sum(need) + n_extra


def as_table(lists, width):
    t = np.full((len(lists), max(width, 1)), -1, dtype=np.int32)
    for i, l in enumerate(lists):
        t[i, :len(l)] = l
    return t


def lfm3_attention(first):
    """plain_lfm3.attention with a window beside which the first positions stay visible."""
    import plain_lfm3 as P

    def part(h, p, T, *, nh, nkv, hd, eps, theta, rope_dim, window=0, gate=False, rnd=P.identity, pos0=0, freq_factors=None):
        pos = torch.arange(pos0, pos0 + T)
        heads = lambda name, n: rnd(h @ p[name].T).view(T, n, hd)
        turn = lambda x, w: rnd(P.rope(P.rms_norm(x, p[w], eps), pos, rope_dim, theta, freq_factors=freq_factors))
        q, k = turn(heads("q_proj.weight", nh), "q_layernorm.weight"), turn(heads("k_proj.weight", nkv), "k_layernorm.weight")
        out = attention(q, k, heads("v_proj.weight", nkv), pos, window, first, 1.0 / math.sqrt(hd))[0]
        if gate:
            out = out * P.sigmoid(rnd(h @ p["gate_proj.weight"].T))[:, :, None]
        return rnd(out.reshape(T, nh * hd)) @ p["out_proj.weight"].T
    return part
