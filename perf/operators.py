"""The operators of the paged key/value cache that is held in 8 bits: what their speed and their results are measured on.

* "tables": a step's tables from request lengths, on the GPU: where every row lies, which pages every request has, with
  pages for what does not fit its last page taken from a stack of free ones.
* "store": the rows [q | k | v] of a step rotated, q handed on, k and v rounded to e4m3 into the pages, with one
  power-of-two scale for each page and head, k and v apart.  A page that held tokens already keeps them: where the new
  ones need a larger scale its older numbers are brought to it.
* "attention": causal grouped-query attention over those pages, single tokens and prompts.

A sequence has `held` tokens in the cache and brings `new` ones; both are spread between the case's bounds and belong to
the case.  Values come from the seed.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda:0"
PAGE = 64
LARGEST, LOWEST_EXPONENT, HIGHEST_EXPONENT = 448.0, -126, 120     # of e4m3; of a page's scale
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def _case(op, seqs, new, held, heads=(28, 4, 128), rot=None, window=0, dtype="bfloat16", name=None):
    c = dict(op=op, seqs=seqs, new_shortest=new[0], new_longest=new[1], held_shortest=held[0], held_longest=held[1])
    if op != "tables":
        c.update(q_heads=heads[0], kv_heads=heads[1], head_dim=heads[2], dtype=dtype)
    if op == "store":
        c.update(rot=heads[2] if rot is None else rot)
    if op == "attention":
        c.update(window=window)
    return dict(c, name=name) if name else c


def listed():
    return [
        # the benchmark's batch of eight conversations, a token each: nothing but latency
        _case("tables", 8, (1, 1), (1000, 2900), name="tables_b8"),
        # a busy server: first and further turns of many conversations together, most of them long
        _case("tables", 256, (1, 1024), (0, 8192), name="tables_turns_b256"),
        # one user, a small model, an odd place in the page
        _case("store", 1, (1, 1), (333, 333), (12, 2, 128), name="store_b1"),
        # the widest decode batch of the benchmark
        _case("store", 64, (1, 1), (1, 500), name="store_b64"),
        # the benchmark's prompt
        _case("store", 1, (2048, 2048), (0, 0), name="store_prompt_2048"),
        # further turns of unequal length in the 32-bit path, half of every head rotated
        _case("store", 12, (1, 700), (0, 300), (16, 4, 128), rot=64, dtype="float32", name="store_turns_f32"),
        # one user, a small model, a short conversation of odd length
        _case("attention", 1, (1, 1), (333, 333), (12, 2, 128), name="attn_b1"),
        # the benchmark's batch of eight conversations
        _case("attention", 8, (1, 1), (1000, 2900), name="attn_b8"),
        # many conversations, short and long: the cache's bytes
        _case("attention", 64, (1, 1), (512, 8191), name="attn_b64"),
        # two documents of the longest length that the model takes
        _case("attention", 2, (1, 1), (30000, 32767), name="attn_long"),
        # the benchmark's prompt
        _case("attention", 1, (2048, 2048), (0, 0), name="attn_prompt_2048"),
        # a further turn in the 32-bit path
        _case("attention", 2, (40, 100), (200, 900), (12, 2, 128), dtype="float32", name="attn_turns_f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _two(rng, lo, hi):
    a, b = _log(rng, lo, hi), _log(rng, lo, hi)
    return min(a, b), max(a, b)


# query heads, key/value heads, head size: of the benchmark's models and of the tests' small ones
HEADS = [(28, 4, 128), (28, 4, 128), (12, 2, 128), (16, 4, 128), (6, 1, 64), (6, 1, 32), (5, 5, 48), (4, 2, 16)]


def draw(rng):
    op = rng.choice(["tables", "store", "store", "attention", "attention", "attention"])
    kind = rng.choice(["decode", "prompt"])
    if op == "tables":
        seqs = _log(rng, 1, 256)
        held = _two(rng, 1, 8192)
        return _case(op, seqs, (1, 1) if kind == "decode" else (rng.randint(0, 1), _log(rng, 2, 1024)), (rng.choice([0, held[0]]), held[1]))
    heads = rng.choice(HEADS)
    dtype = rng.choice(["bfloat16"] * 4 + ["float32"])
    if op == "store":
        rot = rng.choice([heads[2], heads[2], heads[2] // 2])
        if kind == "decode":
            held = _two(rng, 1, 600)
            return _case(op, _log(rng, 1, 64), (1, 1), (rng.choice([0, held[0]]), held[1]), heads, rot, dtype=dtype)
        seqs = _log(rng, 1, 16)
        new = _two(rng, 1, 2048 // seqs)
        return _case(op, seqs, new, (0, rng.choice([0, _log(rng, 1, 400)])), heads, rot, dtype=dtype)
    window = rng.choice([0, 0, 0, 40, 1024])
    if kind == "decode":
        seqs = _log(rng, 1, 64)
        held = _two(rng, 1, min(32767, 262144 // seqs))
        if dtype == "float32":
            held = (min(held[0], 4096), min(held[1], 4096))
        n = rng.choice([1, 1, 1, 2])
        return _case(op, seqs, (1, n), held, heads, window=window, dtype=dtype)
    seqs = _log(rng, 1, 8)
    new = _two(rng, 3, (2048 if dtype == "bfloat16" else 512) // seqs)
    return _case(op, seqs, new, (0, rng.choice([0, _log(rng, 16, 2048 // seqs)])), heads, window=window, dtype=dtype)


def _lengths(case):
    """(new, held) of every sequence, the case's bounds among them."""
    n = case["seqs"]
    rng = random.Random("lengths %d %d %d %d %d" % (n, case["new_shortest"], case["new_longest"], case["held_shortest"], case["held_longest"]))

    def spread(lo, hi):
        if n == 1:
            return [hi]
        got = [lo, hi] + [rng.randint(lo, hi) for _ in range(n - 2)]
        rng.shuffle(got)
        return got

    return spread(case["new_shortest"], case["new_longest"]), spread(case["held_shortest"], case["held_longest"])


def _pages(tokens):
    return -(-tokens // PAGE)


def work(case):
    new, held = _lengths(case)
    rows, total = sum(new), sum(_pages(h + n) for n, h in zip(new, held))
    if case["op"] == "tables":
        old = sum(_pages(h) for h in held)
        # a request's slot, tokens and length in, its row, position and page offsets out; held pages and free ones in, every
        # page out, and into the table where it is new; three numbers a row out
        return {"bytes": 4.0 * (6 * len(new) + old + (total - old) * 2 + total + 3 * rows), "flops": 0.0}
    hq, hkv, hd, out = case["q_heads"], case["kv_heads"], case["head_dim"], DTYPES[case["dtype"]].itemsize
    if case["op"] == "store":
        touched = sum(_pages(h + n) - h // PAGE for n, h in zip(new, held) if n)
        return {"bytes": float(rows * (hq + 2 * hkv) * hd * 4 + rows * case["rot"] * 4 + rows * hq * hd * out + rows * 2 * hkv * hd
                               + touched * 2 * hkv * 4), "flops": float(rows * (hq + hkv) * case["rot"] * 3)}
    window = case["window"]
    reach = lambda p: min(p + 1, window) if window else p + 1                                                # noqa: E731
    keys = sum(min(h + n, window + n - 1) if window else h + n for n, h in zip(new, held) if n)
    pairs = 0
    for n, h in zip(new, held):
        if window and h + n > window:
            pairs += sum(reach(p) for p in range(h, h + n))
        else:
            pairs += n * h + n * (n + 1) // 2
    return {"bytes": float(keys * 2 * hkv * hd + _pages(keys) * 2 * hkv * 4 + rows * hq * hd * 2 * out), "flops": 4.0 * pairs * hq * hd}


# ------------------------------------------------------------------------------------------------ states
class _Group:
    def __init__(self, page_off, page_ids):
        self.page_off, self.page_ids, self.page_size = page_off, page_ids, PAGE


class _Plan:
    """A step's plan as a program keeps it for all layers of a step."""

    def __init__(self, new, held, page_lists):
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)                                    # noqa: E731
        row0, off = [0], [0]
        for n, p in zip(new, page_lists):
            row0.append(row0[-1] + n)
            off.append(off[-1] + len(p))
        self.n_seqs, self.n_rows, self.max_new = len(new), row0[-1], max(new)
        self.max_len = max(n + h for n, h in zip(new, held))
        self.seq_row0, self.seq_pos0 = i32(row0), i32(held)
        seq = torch.repeat_interleave(torch.arange(len(new), device=DEVICE), torch.tensor(new, device=DEVICE))
        self.row_seq = seq.int()
        self.row_pos = (torch.arange(self.n_rows, device=DEVICE) - self.seq_row0[seq] + self.seq_pos0[seq]).int()
        self.groups = [_Group(i32(off), i32([p for l in page_lists for p in l]))]
        self._scratch = None

    def scratch(self, nbytes, device):
        if nbytes <= 0:
            return None
        if self._scratch is None or self._scratch.numel() < nbytes:
            self._scratch = torch.empty(nbytes, dtype=torch.uint8, device=device)
        return self._scratch


def _exponents(largest):
    """The smallest e with largest <= 448 * 2^e, in the range of a page's scale."""
    m, x = torch.frexp(largest)
    return (x - torch.where(m <= 0.875, 9, 8)).clamp(LOWEST_EXPONENT, HIGHEST_EXPONENT)


def _filled(n_pages, kv_heads, head_dim, g):
    """Pages as conversations leave them: keys with a few large channels, values of unequal size from head to head."""
    x = torch.randn(n_pages, 2, kv_heads, PAGE, head_dim, generator=g, device=DEVICE)
    size = torch.ones(2, kv_heads, 1, head_dim, device=DEVICE)
    size[0, :, :, :: max(2, head_dim // 4)] = 3.0
    size[1] *= torch.linspace(0.3, 2.0, kv_heads, device=DEVICE).view(kv_heads, 1, 1)
    x *= size
    scale = torch.exp2(_exponents(x.abs().amax((3, 4))).float())
    return (x / scale[..., None, None]).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    new, held = _lengths(case)
    rng = random.Random(seed)
    if case["op"] == "tables":
        n, wide = len(new), _pages(max(h + t for t, h in zip(new, held)))
        n_slots = 2 * n + 1
        total = sum(_pages(h + t) for t, h in zip(new, held))
        ids = list(range(total + 16))
        rng.shuffle(ids)
        slots = rng.sample(range(n_slots), n)
        table, lengths, at = torch.full((n_slots, wide), -1, dtype=torch.int32), torch.zeros(n_slots, dtype=torch.int32), 0
        for s, h in zip(slots, held):
            lengths[s] = h
            table[s, :_pages(h)] = torch.tensor(ids[at:at + _pages(h)], dtype=torch.int32)
            at += _pages(h)
        free = ids[at:]
        i32 = lambda v: torch.as_tensor(v, dtype=torch.int32).to(DEVICE)                                     # noqa: E731
        return dict(op="tables", slots=i32(slots), new=i32(new), lengths=i32(lengths), table=i32(table), free=i32(free + [-1] * at),
                    n_free=i32([len(free)]), rows=sum(new) + 3, pages=total, max_new=max(new), max_len=wide * PAGE, out=None)
    hq, hkv, hd, dtype = case["q_heads"], case["kv_heads"], case["head_dim"], DTYPES[case["dtype"]]
    counts = [_pages(h + t) for t, h in zip(new, held)]
    ids = list(range(sum(counts) + 1))
    rng.shuffle(ids)
    lists, at = [], 0
    for c in counts:
        lists.append(ids[at:at + c])
        at += c
    plan = _Plan(new, held, lists)
    cache, scales = _filled(len(ids), hkv, hd, g)
    s = dict(op=case["op"], plan=plan, cache=cache, scales=scales, q_heads=hq, kv_heads=hkv, head_dim=hd)
    if case["op"] == "store":
        rot = case["rot"]
        s["rot"], s["qkv"] = rot, torch.randn(plan.n_rows, (hq + 2 * hkv) * hd, generator=g, device=DEVICE) * 1.5
        inv = torch.arange(0, rot, 2, device=DEVICE, dtype=torch.float64).div(-rot).mul(math.log(1e6)).exp()
        theta = plan.row_pos.double()[:, None] * inv
        s["angles"] = torch.cat([theta.cos(), theta.sin()], 1).float()
        s["q_out"] = torch.empty(plan.n_rows, hq, hd, dtype=dtype, device=DEVICE)
        return s
    s["window"], s["scale"] = case["window"], hd ** -0.5
    s["q"] = torch.randn(plan.n_rows, hq, hd, generator=g, device=DEVICE).to(dtype)
    s["out"] = torch.empty(plan.n_rows, hq * hd, dtype=dtype, device=DEVICE)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _tables(s):
    slots, new, table, free = s["slots"].long(), s["new"].long(), s["table"], s["free"]
    length = s["lengths"][slots].long()
    zero = torch.zeros(1, dtype=torch.long, device=slots.device)
    have, total = (length + PAGE - 1) // PAGE, (length + new + PAGE - 1) // PAGE
    row0, off, taken = (torch.cat([zero, v.cumsum(0)]) for v in (new, total, total - have))
    row = torch.arange(s["rows"], device=slots.device)
    inside = row < row0[-1]
    seq = torch.searchsorted(row0, row, right=True).sub(1).clamp(max=slots.numel() - 1)
    pos = length[seq] + row - row0[seq]
    page = torch.arange(s["pages"], device=slots.device)
    there = page < off[-1]
    owner = torch.searchsorted(off, page, right=True).sub(1).clamp(max=slots.numel() - 1)
    place = page - off[owner]
    fresh = place >= have[owner]
    nth = (taken[owner] + place - have[owner]).clamp(min=0)
    ids = torch.where(fresh, free[(s["n_free"] - 1 - nth).clamp(min=0)], table[slots[owner], place.clamp(max=table.shape[1] - 1)])
    ids = torch.where(there, ids, -1)
    at = torch.where(there & fresh, place, table.shape[1])          # a column beyond the table for what is not written
    table.copy_(torch.cat([table, table[:, :1]], 1).index_put((slots[owner], at), ids)[:, :-1])
    where = ids[(off[seq] + pos // PAGE).clamp(max=s["pages"] - 1)] * PAGE + pos % PAGE
    i32 = lambda v: v.to(torch.int32)                                                                        # noqa: E731
    return dict(seq_row0=i32(row0), seq_pos0=i32(length), row_seq=i32(torch.where(inside, seq, 0)), row_pos=i32(torch.where(inside, pos, -1)),
                row_slot=i32(torch.where(inside, where, -1)), page_off=i32(off), page_ids=ids, table=table)


def _store(s):
    plan, hq, hkv, hd, rot = s["plan"], s["q_heads"], s["kv_heads"], s["head_dim"], s["rot"]
    g, cache, scales = plan.groups[0], s["cache"], s["scales"]
    x = s["qkv"].view(plan.n_rows, hq + 2 * hkv, hd)
    cos, sin = s["angles"][:, None, :rot // 2], s["angles"][:, None, rot // 2:]
    qk = x[:, :hq + hkv]
    a, b = qk[..., :rot // 2], qk[..., rot // 2:rot]
    qk = torch.cat([a * cos - b * sin, a * sin + b * cos, qk[..., rot:]], -1)
    s["q_out"].copy_(qk[:, :hq])
    kv = torch.stack([qk[:, hq:], x[:, hq + hkv:]], 1)              # [row, k|v, head, value]
    # the pages that get a row, at most `n` of every sequence
    n = (plan.max_new + 2 * PAGE - 2) // PAGE
    pos0, count = plan.seq_pos0.long(), (plan.seq_row0[1:] - plan.seq_row0[:-1]).long()
    nth = pos0[:, None] // PAGE + torch.arange(n, device=x.device)
    used = (nth * PAGE < (pos0 + count)[:, None]) & (count > 0)[:, None]
    spare = cache.shape[0]                                          # a page of their own for places without one
    ids = torch.where(used, g.page_ids[(g.page_off[:-1, None] + nth).clamp(max=g.page_ids.numel() - 1)].long(), spare).view(-1)
    seq, pos = plan.row_seq.long(), plan.row_pos.long()
    mine = seq * n + pos // PAGE - pos0[seq] // PAGE                # a row's page among them
    e = torch.full((ids.numel(), 2, hkv), LOWEST_EXPONENT, dtype=torch.int32, device=x.device)
    e = e.index_reduce(0, mine, _exponents(kv.abs().amax(3)).int(), "amax")
    older = (pos0[:, None] > nth * PAGE).view(-1)
    padded = torch.cat([scales, torch.ones_like(scales[:1])])
    before = padded[ids]
    e = torch.where(older[:, None, None], torch.maximum(e, torch.frexp(before)[1] - 1), e)
    scale = torch.exp2(e.float())
    held = torch.cat([cache.view(torch.uint8), cache[:1].view(torch.uint8)])[ids].view(torch.float8_e4m3fn).float()
    held = held * (before / scale)[..., None, None]
    keep = (torch.arange(PAGE, device=x.device) < (pos0[:, None] - nth * PAGE).view(-1, 1))     # tokens from earlier steps
    stale = cache.view(torch.uint8)[ids.clamp(max=spare - 1)]
    page = torch.where(keep[:, None, None, :, None], held.to(torch.float8_e4m3fn).view(torch.uint8), stale)
    rounded = (kv / scale[mine][..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
    page = page.permute(0, 3, 1, 2, 4).index_put((mine, pos % PAGE), rounded).permute(0, 2, 3, 1, 4)
    cache.copy_(torch.cat([cache.view(torch.uint8), cache[:1].view(torch.uint8)]).index_copy(0, ids, page)[:-1].view(torch.float8_e4m3fn))
    scales.copy_(padded.index_copy(0, ids, scale)[:-1])
    return dict(q=s["q_out"], cache=cache, scales=scales)


def _attention(s):
    plan, hq, hkv, hd = s["plan"], s["q_heads"], s["kv_heads"], s["head_dim"]
    g, most = plan.groups[0], _pages(plan.max_len)
    group, n_seqs, q = hq // hkv, plan.n_seqs, s["q"]
    nth = torch.arange(most, device=q.device)
    there = nth < (g.page_off[1:] - g.page_off[:-1])[:, None]
    ids = torch.where(there, g.page_ids[(g.page_off[:-1, None] + nth).clamp(max=g.page_ids.numel() - 1)], 0).long()
    pages = s["cache"].view(torch.uint8)[ids].view(torch.float8_e4m3fn).float() * s["scales"][ids][..., None, None]
    k, v = (pages[:, :, i].transpose(1, 2).reshape(n_seqs, hkv, most * PAGE, hd) for i in (0, 1))
    new = torch.arange(plan.max_new, device=q.device)
    rows = (plan.seq_row0[:-1, None] + new).clamp(max=plan.n_rows - 1).long()
    qs = q[rows].float().view(n_seqs, plan.max_new, hkv, group, hd).permute(0, 2, 1, 3, 4).reshape(n_seqs, hkv, -1, hd)
    scores = torch.matmul(qs, k.transpose(2, 3)).mul_(s["scale"]).view(n_seqs, hkv, plan.max_new, group, -1)
    at, key = (plan.seq_pos0[:, None] + new)[:, :, None], torch.arange(most * PAGE, device=q.device)
    seen = key <= at
    if s["window"]:
        seen = seen & (key > at - s["window"])
    scores.masked_fill_(~seen[:, None, :, None], -math.inf)
    p = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(p.view(n_seqs, hkv, plan.max_new * group, -1), v).view(n_seqs, hkv, plan.max_new, group, hd)
    o = (o / p.sum(-1, keepdim=True)).permute(0, 2, 1, 3, 4).reshape(n_seqs, plan.max_new, hq * hd)
    seq = plan.row_seq.long()
    s["out"].copy_(o[seq, (plan.row_pos - plan.seq_pos0[seq]).long()])
    return s["out"]


def run(s):
    if own:
        from sonicboom_b200 import ops
        if s["op"] == "tables":
            if s["out"] is None:
                s["out"] = ops.PageTables(s["slots"].numel(), s["rows"], s["pages"], DEVICE)
            t = ops.page_tables(s["slots"], s["new"], s["lengths"], s["table"], s["free"], s["n_free"], s["out"], s["max_new"], s["max_len"])
            return dict(seq_row0=t.seq_row0, seq_pos0=t.seq_pos0, row_seq=t.row_seq, row_pos=t.row_pos, row_slot=t.row_slot,
                        page_off=t.page_off, page_ids=t.page_ids, table=s["table"])
        if s["op"] == "store":
            ops.rope_store_e4m3(s["qkv"], s["q_heads"], s["kv_heads"], s["head_dim"], s["rot"], s["angles"], s["plan"], 0, s["cache"],
                                s["scales"], s["q_out"])
            return dict(q=s["q_out"], cache=s["cache"], scales=s["scales"])
        return ops.attention_e4m3(s["q"], s["out"], s["plan"], 0, s["cache"], s["scales"], s["q_heads"], s["kv_heads"], s["head_dim"],
                                  s["window"], s["scale"])
    return {"tables": _tables, "store": _store, "attention": _attention}[s["op"]](s)


# ------------------------------------------------------------------------------------------------ in 64 bits
def _to_e4m3(x):
    """x rounded to the nearest e4m3 number, in 64 bits: three bits behind the first one, none below 2^-9."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    if case["op"] == "tables":
        return None                                                  # whole numbers, which have to be equal
    s = prepare(case, seed)
    new, held = _lengths(case)
    plan, hq, hkv, hd = s["plan"], s["q_heads"], s["kv_heads"], s["head_dim"]
    off, ids = plan.groups[0].page_off.tolist(), plan.groups[0].page_ids.tolist()
    if case["op"] == "store":
        cache, scales, half = s["cache"].double(), s["scales"].double(), s["rot"] // 2
        q, at = [], 0
        for i, (n, h) in enumerate(zip(new, held)):
            if n == 0:
                continue
            x = s["qkv"][at:at + n].double().view(n, -1, hd)
            angle = s["angles"][at:at + n].double()
            at += n
            turn = torch.complex(angle[:, :half], angle[:, half:])[:, None]
            y = torch.complex(x[..., :half], x[..., half:2 * half]) * turn
            y = torch.cat([y.real, y.imag, x[..., 2 * half:]], 2)
            q.append(y[:, :hq])
            kv = torch.stack([y[:, hq:hq + hkv], x[:, hq + hkv:]]).permute(1, 0, 2, 3)
            for j in range(h // PAGE, _pages(h + n)):
                lo, hi = max(h, j * PAGE), min(h + n, (j + 1) * PAGE)
                page, old = ids[off[i] + j], lo - j * PAGE
                part = kv[lo - h:hi - h].permute(1, 2, 0, 3)
                need = torch.exp2(torch.ceil(torch.log2((part.abs().amax((2, 3)) / LARGEST).clamp(min=2.0 ** LOWEST_EXPONENT))))
                scale = torch.maximum(need, scales[page]) if old else need
                cache[page, :, :, :old] = _to_e4m3(cache[page, :, :, :old] * (scales[page] / scale)[..., None, None])
                cache[page, :, :, old:old + hi - lo] = _to_e4m3(part / scale[..., None, None])
                scales[page] = scale
        return dict(q=torch.cat(q), cache=cache, scales=scales)
    out, at = [], 0
    for i, (n, h) in enumerate(zip(new, held)):
        if n == 0:
            continue
        mine = torch.tensor(ids[off[i]:off[i + 1]], device=DEVICE)
        kv = s["cache"].view(torch.uint8)[mine].view(torch.float8_e4m3fn).double() * s["scales"][mine].double()[..., None, None]
        kv = kv.permute(1, 2, 0, 3, 4).reshape(2, hkv, -1, hd)[:, :, :h + n].repeat_interleave(hq // hkv, 1)
        q = s["q"][at:at + n].double().transpose(0, 1)
        at += n
        score = q @ kv[0].transpose(1, 2) * s["scale"]
        back = torch.arange(h, h + n, device=DEVICE)[:, None] - torch.arange(h + n, device=DEVICE)
        hidden = back < 0
        if s["window"]:
            hidden = hidden | (back >= s["window"])
        weight = torch.softmax(score.masked_fill(hidden, -math.inf), 2)
        out.append((weight @ kv[1]).transpose(0, 1).reshape(n, hq * hd))
    return torch.cat(out)
