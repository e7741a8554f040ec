"""A plain, slow form of the paged cache in 8 bits on the host: numbers in 64 bits, one token after another, pages as lists.

What it is compared with bit for bit is exact here: e4m3 numbers and scales are small dyadic fractions, the rotation is done
in float32 with every product and sum rounded on its own, and rounding to e4m3 goes by the definition."""
import math

import torch

PAGE = 64


def round_e4m3(x):
    """float64 to the nearest e4m3 number, ties to even; infinities and NaN to NaN."""
    fine = torch.isfinite(x)
    v = torch.where(fine, x, torch.zeros_like(x))
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.where(fine, torch.round(v / step) * step, torch.full_like(x, math.nan))


def exponent_for(largest: float) -> int:
    """The smallest e >= -126 with largest <= 448 * 2^e."""
    e = -126
    while largest > 448.0 * 2.0 ** e:
        e += 1
    return e


def rotate(x, cos, sin):
    """[..., hd] float32 by cos, sin [rot / 2]: every product and sum rounded to float32."""
    half = cos.shape[-1]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., 2 * half:]], -1)


class PlainCache:
    """Pages of e4m3 numbers (float64) with a scale for each page, k|v and head."""

    def __init__(self, n_pages, n_kv_heads, hd, page=PAGE):
        self.numbers = torch.zeros(n_pages, 2, n_kv_heads, page, hd, dtype=torch.float64)
        self.scales = torch.zeros(n_pages, 2, n_kv_heads, dtype=torch.float64)
        self.page = page

    def store(self, pages, pos0, kv):
        """kv [n, k|v, head, hd] float32 of the positions pos0 ... of a sequence with these pages (-1, or beyond the list: none)."""
        kv, n_pages = kv.double(), self.numbers.shape[0]
        at = 0
        while at < kv.shape[0]:
            i, place = divmod(pos0 + at, self.page)
            n = min(self.page - place, kv.shape[0] - at)
            if i < len(pages) and 0 <= pages[i] < n_pages:
                p = pages[i]
                for kind in range(2):
                    for h in range(kv.shape[2]):
                        x = kv[at:at + n, kind, h]
                        e = exponent_for(float(torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).max()))
                        if place:
                            before = int(math.log2(float(self.scales[p, kind, h])))
                            if e > before:
                                old = self.numbers[p, kind, h, :place]
                                self.numbers[p, kind, h, :place] = round_e4m3(old * 2.0 ** (before - e))
                            e = max(e, before)
                        self.scales[p, kind, h] = 2.0 ** e
                        self.numbers[p, kind, h, place:place + n] = round_e4m3(x * 2.0 ** -e)
            at += n

    def keys_values(self, pages, n):
        """[k|v, head, n, hd] in 64 bits of a sequence's first n positions."""
        picked = torch.tensor([max(p, 0) for p in pages[:-(-n // self.page)]])
        v = self.numbers[picked] * self.scales[picked][..., None, None]
        return v.permute(1, 2, 0, 3, 4).reshape(2, v.shape[2], -1, v.shape[4])[:, :, :n]


def attend(q, kv, pos0, window, scale):
    """q [n, heads, hd], kv [k|v, kv head, keys, hd], all 64 bits: (result [n, heads, hd], what its error is measured by).

    The second is (sum_j p_j |v_j|, the largest sum_d |q_d k_jd| over the keys seen): errors of weights scale with the first, errors
    of scores with the second."""
    n, hq, hd = q.shape
    group = hq // kv.shape[1]
    k, v = kv[0].repeat_interleave(group, 0), kv[1].repeat_interleave(group, 0)
    pos = torch.arange(pos0, pos0 + n)
    key = torch.arange(k.shape[1])
    seen = key <= pos[:, None]
    if window:
        seen &= key > pos[:, None] - window
    s = torch.einsum("nhd,hkd->hnk", q, torch.nan_to_num(k)) * scale
    s = torch.where(torch.isnan(k).any(-1)[:, None, :], math.nan, s).masked_fill(~seen, -math.inf)
    p = torch.softmax(s, -1)
    out = torch.zeros(hq, n, hd, dtype=torch.float64)
    size = torch.zeros_like(out)
    for i in range(n):                                    # keys that a row does not see take no part, whatever they hold
        out[:, i] = torch.einsum("hk,hkd->hd", p[:, i, seen[i]], v[:, seen[i]])
        size[:, i] = torch.einsum("hk,hkd->hd", p[:, i, seen[i]], v[:, seen[i]].abs())
    dots = torch.einsum("nhd,hkd->hnk", q.abs(), torch.nan_to_num(k).abs()).masked_fill(~seen, 0).amax(-1)
    return out.transpose(0, 1), size.transpose(0, 1), dots.transpose(0, 1)


def tolerance(out, size, dots, scale, hd, keys, dtype):
    """How far a row may be off, by arithmetic.  A score is a sum of hd products in 32 bits times scale: off by at most
    (hd + 3) 2^-24 scale sum|q k|, which moves weights (and their sum) by that much, relatively, and the exponential by 2^-21 more.
    Sums over the keys in 32 bits: at most keys 2^-24 of sum p|v|, and as much again for the weights' sum.  bfloat16 rows: weights
    rounded to at least 8 bits (half a step, 2^-8, when the kernel multiplies bfloat16 weights) and the result to bfloat16 (2^-8
    of it)."""
    by_scores = 2 * (hd + 3) * 2.0 ** -24 * abs(scale) * dots[..., None] + 2.0 ** -20
    by_sums = 2 * (keys + 8) * 2.0 ** -24
    if dtype == torch.bfloat16:
        return 2.0 ** -8 * out.abs() + (2.0 ** -8 + by_scores + by_sums) * size + 1e-30
    return 2.0 ** -23 * out.abs() + (by_scores + by_sums) * size + 1e-30


class PlainPages:
    """`page_tables` and its companions with lists: lengths, page lists, a stack of free pages."""

    def __init__(self, n_slots, width, free, page=PAGE):
        self.lengths, self.pages, self.free, self.width, self.page = [0] * n_slots, [[] for _ in range(n_slots)], list(free), width, page

    def count(self, tokens):
        return -(-tokens // self.page)

    def status(self, slots, new, max_rows, max_pages, max_new, max_len):
        bad, rows, total, need, named = 0, 0, 0, 0, set()
        for s, n in zip(slots, new):
            if not 0 <= s < len(self.lengths) or n < 0 or s in named:
                bad |= 1
                continue
            named.add(s)
            length = self.lengths[s] + n
            if n > max_new or length > max_len or self.count(length) > self.width:
                bad |= 2
                continue
            rows, total, need = rows + n, total + self.count(length), need + self.count(length) - self.count(self.lengths[s])
        return bad | (4 if rows > max_rows else 0) | (8 if total > max_pages else 0) | (16 if need > len(self.free) else 0)

    def tables(self, slots, new):
        """(row0, pos0, row_seq, row_pos, row_slot, page lists); takes nothing yet."""
        top, lists, row0, rows = len(self.free), [], [0], []
        for i, (s, n) in enumerate(zip(slots, new)):
            mine = list(self.pages[s])
            while len(mine) < self.count(self.lengths[s] + n):
                top -= 1
                mine.append(self.free[top])
            lists.append(mine)
            row0.append(row0[-1] + n)
            for pos in range(self.lengths[s], self.lengths[s] + n):
                rows.append((i, pos, mine[pos // self.page] * self.page + pos % self.page))
        return row0, [self.lengths[s] for s in slots], rows, lists

    def advance(self, slots, new):
        _, _, _, lists = self.tables(slots, new)
        taken = sum(len(m) - len(self.pages[s]) for s, m in zip(slots, lists))
        for s, n, mine in zip(slots, new, lists):
            self.pages[s], self.lengths[s] = mine, self.lengths[s] + n
        del self.free[len(self.free) - taken:]

    def release(self, slots):
        for s in dict.fromkeys(slots):
            if 0 <= s < len(self.lengths):
                self.free += self.pages[s]
                self.pages[s], self.lengths[s] = [], 0
