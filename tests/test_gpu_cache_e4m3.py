"""The 8-bit cache's kernels against the plain form in 64 bits: what they store bit for bit, what they attend to within the
tolerance that arithmetic gives, tables exactly; then all of them together in a replayed graph."""
import math
import random

import pytest
import torch

import plain_cache_e4m3 as plain
from sonicboom_b200 import ops
from sonicboom_b200.cache import DevicePages

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
PAGE = 64


class Plan:
    """A step's plan from lists: positions and pages of sequences that bring new[i] tokens each."""

    def __init__(self, new, pos0, lists, spare_rows=0):
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)                   # noqa: E731
        self.n_seqs, self.n_rows = len(new), sum(new) + spare_rows
        self.max_new, self.max_len = max(max(new), 1), max(max(p + n for p, n in zip(pos0, new)), 1)
        row0, off = [0], [0]
        for n, pages in zip(new, lists):
            row0.append(row0[-1] + n)
            off.append(off[-1] + len(pages))
        self.seq_row0, self.seq_pos0 = i32(row0), i32(pos0)
        self.row_seq = i32([i for i, n in enumerate(new) for _ in range(n)] + [0] * spare_rows)
        self.row_pos = i32([p + j for p, n in zip(pos0, new) for j in range(n)] + [-1] * spare_rows)
        self.groups = [ops.TableGroup(i32(off), i32([p for pages in lists for p in pages] or [0]), PAGE)]
        self._scratch = None

    def scratch(self, nbytes, device):
        if nbytes <= 0:
            return None
        if self._scratch is None or self._scratch.numel() < nbytes:
            self._scratch = torch.empty(nbytes, dtype=torch.uint8, device=device)
        return self._scratch


def shuffled_lists(rng, lengths, spare=2):
    ids = list(range(sum(-(-n // PAGE) for n in lengths) + spare))
    rng.shuffle(ids)
    out, at = [], 0
    for n in lengths:
        out.append(ids[at:at + -(-n // PAGE)])
        at += -(-n // PAGE)
    return out, len(ids)


def device_cache(n_pages, hkv, hd):
    """Pages full of what other sequences left behind: any byte, NaN among them, and any scale."""
    g = torch.Generator().manual_seed(n_pages + hkv + hd)
    numbers = torch.randint(0, 256, (n_pages, 2, hkv, PAGE, hd), generator=g, dtype=torch.uint8)
    scales = torch.exp2(torch.randint(-126, 121, (n_pages, 2, hkv), generator=g).float())
    return numbers.to(DEV).view(torch.float8_e4m3fn), scales.to(DEV)


def fill(cache, oracle):
    """The plain cache's pages in the device's form (its numbers are e4m3 numbers: nothing is rounded)."""
    return oracle.numbers.float().to(torch.float8_e4m3fn).to(DEV), oracle.scales.float().to(DEV)


def rows_of(n, hq, hkv, hd, g, size=1.0):
    x = torch.randn(n, hq + 2 * hkv, hd, generator=g) * size
    x[:, hq:hq + hkv, ::7] *= 6.0                       # keys with large channels
    return x


# ------------------------------------------------------------------------------------------------ store
STEPS = [  # what every sequence brings, step by step: first tokens, page ends, single tokens, nothing, several pages
    [[1, 64, 5, 0, 130], [1, 1, 59, 3, 0], [62, 0, 1, 61, 1], [1, 129, 64, 1, 70]],
    [[333], [1], [1], [50], [1]],
    [[3, 8, 1, 0], [5, 2, 8, 1], [60, 62, 50, 70], [1, 2, 3, 4], [8, 8, 8, 8]],
]


@pytest.mark.parametrize("hq,hkv,hd,rot", [(4, 2, 128, 128), (6, 1, 64, 32), (5, 5, 48, 48), (2, 2, 16, 16), (3, 1, 256, 128), (2, 1, 22, 8), (4, 2, 96, 0)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("steps", STEPS)
def test_store_bit_for_bit(hq, hkv, hd, rot, dtype, steps):
    g, rng = torch.Generator().manual_seed(hd + rot), random.Random(hd)
    n_seqs = len(steps[0])
    lists, n_pages = shuffled_lists(rng, [sum(s[i] for s in steps) for i in range(n_seqs)])
    oracle = plain.PlainCache(n_pages, hkv, hd)
    cache, scales = device_cache(n_pages, hkv, hd)
    before = cache.view(torch.uint8).clone()
    pos0 = [0] * n_seqs
    for k, new in enumerate(steps):
        plan = Plan(new, pos0, lists, spare_rows=2)
        size = 10.0 ** rng.uniform(-3, 3) if k else 0.01                       # later steps larger or smaller than what a page holds
        x = rows_of(plan.n_rows, hq, hkv, hd, g, size)
        angle = torch.randn(plan.n_rows, max(rot // 2, 1), generator=g)
        angles = torch.cat([angle.cos(), angle.sin()], 1)[:, :rot] if rot else None
        q_out = torch.full((plan.n_rows, hq, hd), 7.0, dtype=dtype, device=DEV)
        ops.rope_store_e4m3(x.view(plan.n_rows, -1).to(DEV), hq, hkv, hd, rot, angles.to(DEV) if rot else None, plan, 0, cache, scales, q_out)
        turned = x.clone()
        if rot:
            turned[:, :hq + hkv] = plain.rotate(x[:, :hq + hkv], angles[:, None, :rot // 2], angles[:, None, rot // 2:])
        rows = sum(new)
        assert torch.equal(q_out[:rows].cpu(), turned[:rows, :hq].to(dtype))
        assert bool((q_out[rows:] == 7.0).all())                                # rows behind the last sequence
        at = 0
        for i, n in enumerate(new):
            oracle.store(lists[i], pos0[i], torch.stack([turned[at:at + n, hq:hq + hkv], turned[at:at + n, hq + hkv:]], 1))
            at += n
        pos0 = [p + n for p, n in zip(pos0, new)]
        numbers, kept = cache.float().cpu().double(), scales.cpu().double()
        for i in range(n_seqs):
            for j, page in enumerate(lists[i][:-(-pos0[i] // PAGE)]):
                held = min(PAGE, pos0[i] - j * PAGE)
                assert torch.equal(numbers[page, :, :, :held], oracle.numbers[page, :, :, :held]), (k, i, j)
                assert torch.equal(kept[page], oracle.scales[page]), (k, i, j)
    # what nobody wrote is what it was
    mine = torch.zeros(n_pages, PAGE, dtype=torch.bool)
    for i in range(n_seqs):
        for j, page in enumerate(lists[i]):
            mine[page, :max(0, min(PAGE, pos0[i] - j * PAGE))] = True
    same = (cache.view(torch.uint8) == before).cpu().all(-1)
    assert bool(same.permute(0, 3, 1, 2)[~mine].all())


def test_store_of_values_without_a_size():
    """Infinities and NaN are stored as NaN and leave the scale alone; zeros and the smallest values have the lowest scale."""
    hd, hkv = 32, 1
    plan = Plan([4], [0], [[1]])
    cache, scales = device_cache(2, hkv, hd)
    x = torch.zeros(4, 3, hd)
    x[0, 1, :4] = torch.tensor([math.inf, -math.inf, math.nan, 2.5])
    x[1, 1] = 100.0
    x[2, 2, 0] = 1e-40
    x[3, 2, 1] = -3.4028234663852886e38
    q = torch.empty(4, 1, hd, device=DEV)
    ops.rope_store_e4m3(x.view(4, -1).to(DEV), 1, hkv, hd, 0, None, plan, 0, cache, scales, q)
    oracle = plain.PlainCache(2, hkv, hd)
    oracle.store([1], 0, torch.stack([x[:, 1:2], x[:, 2:3]], 1))
    got = cache.float().cpu().double()[1, :, :, :4]
    assert torch.equal(torch.nan_to_num(got, nan=-1e9), torch.nan_to_num(oracle.numbers[1, :, :, :4], nan=-1e9))
    assert torch.equal(scales.cpu().double()[1], oracle.scales[1])
    assert bool(got[0, 0, 0, :3].isnan().all()) and float(scales[1, 0, 0]) == 2.0 ** -2
    # a later token of ordinary size over values that were all but zero
    plan = Plan([1], [4], [[1]])
    y = torch.full((1, 3, hd), 3.0)
    ops.rope_store_e4m3(y.view(1, -1).to(DEV), 1, hkv, hd, 0, None, plan, 0, cache, scales, q[:1])
    oracle.store([1], 4, torch.stack([y[:, 1:2], y[:, 2:3]], 1))
    got = cache.float().cpu().double()[1, :, :, :5]
    assert torch.equal(torch.nan_to_num(got, nan=-1e9), torch.nan_to_num(oracle.numbers[1, :, :, :5], nan=-1e9))


def test_store_without_a_page_writes_nothing_but_q():
    hq, hkv, hd = 2, 1, 64
    lists = [[1, -1, 3], [2], [0, 9999]]                                        # given back; too short a list; no page of this cache
    plan = Plan([3, 10, 66], [64, 60, 60], lists)
    cache, scales = device_cache(5, hkv, hd)
    before, kept = cache.view(torch.uint8).clone(), scales.clone()
    x = rows_of(plan.n_rows, hq, hkv, hd, torch.Generator().manual_seed(1))
    q = torch.empty(plan.n_rows, hq, hd, device=DEV)
    ops.rope_store_e4m3(x.view(plan.n_rows, -1).to(DEV), hq, hkv, hd, 0, None, plan, 0, cache, scales, q)
    assert torch.equal(q.cpu(), x[:, :hq])
    changed = (cache.view(torch.uint8) != before).any(-1).cpu()                 # [page, k|v, head, place]
    places = {(p, s) for p, _, _, s in changed.nonzero().tolist()}
    assert places <= {(2, s) for s in range(64)} | {(0, s) for s in range(64)} and (2, 60) in places and (0, 63) in places
    assert torch.equal(scales[[1, 3, 4]], kept[[1, 3, 4]])


# ------------------------------------------------------------------------------------------------ attention
def attention_case(new, pos0, hq, hkv, hd, dtype, window=0, seed=0, spread=0.0, scale=None, kernel="auto"):
    """Runs the operator on a cache that the plain form filled; compares every row."""
    g, rng = torch.Generator().manual_seed(seed + hd), random.Random(seed)
    lengths = [p + n for p, n in zip(pos0, new)]
    lists, n_pages = shuffled_lists(rng, lengths)
    oracle = plain.PlainCache(n_pages, hkv, hd)
    for pages, n in zip(lists, lengths):
        x = torch.randn(n, 2, hkv, hd, generator=g)
        if spread:                                                              # pages of very unequal scale
            x *= torch.exp2(torch.randint(-int(spread), int(spread) + 1, (-(-n // PAGE),), generator=g).float()).repeat_interleave(PAGE)[:n, None, None, None]
        oracle.store(pages, 0, x)
    cache, scales = fill(None, oracle)
    stale, _ = device_cache(n_pages, hkv, hd)
    held = torch.zeros(n_pages, PAGE, dtype=torch.bool)
    for pages, n in zip(lists, lengths):
        for j, p in enumerate(pages):
            held[p, :min(PAGE, n - j * PAGE)] = True
    keep = held[:, None, None, :, None].to(DEV)
    cache = torch.where(keep, cache.view(torch.uint8), stale.view(torch.uint8)).view(torch.float8_e4m3fn)   # NaN behind the lengths
    if window:                                                                  # pages that no row sees have been given back
        lists = [[-1 if (j + 1) * PAGE <= p - window + 1 else page for j, page in enumerate(pages)] for pages, p in zip(lists, pos0)]
    plan = Plan(new, pos0, lists, spare_rows=1)
    q = torch.randn(plan.n_rows, hq, hd, generator=g).to(dtype)
    out = torch.full((plan.n_rows, hq * hd), 5.0, dtype=dtype, device=DEV)
    scale = hd ** -0.5 if scale is None else scale
    ops.attention_e4m3(q.to(DEV), out, plan, 0, cache, scales, hq, hkv, hd, window, scale, kernel)
    got = out.cpu().double().view(plan.n_rows, hq, hd)
    at = 0
    for pages, p, n in zip(lists, pos0, new):
        if n:
            want, size, dots = plain.attend(q[at:at + n].double(), oracle.keys_values(pages, p + n), p, window, scale)
            far = (got[at:at + n] - want).abs() / plain.tolerance(want, size, dots, scale, hd, p + n, dtype)
            assert float(far.max()) <= 1.0, (n, p, float(far.max()))
        at += n
    assert bool((got[at:] == 5.0).all())                                        # rows behind the last sequence
    return plan, q, out, cache, scales


HEADS = [(28, 4, 128), (12, 2, 128), (6, 1, 64), (5, 5, 48), (4, 2, 16), (4, 4, 80), (3, 1, 256), (8, 2, 112), (2, 1, 24), (4, 1, 22)]


@pytest.mark.parametrize("hq,hkv,hd", HEADS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_of_single_tokens(hq, hkv, hd, dtype):
    attention_case([1, 1, 1, 1, 1, 0, 1, 1], [0, 62, 63, 64, 333, 100, 700, 1], hq, hkv, hd, dtype)


@pytest.mark.parametrize("hq,hkv,hd", HEADS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_of_prompts(hq, hkv, hd, dtype):
    attention_case([70, 1, 0, 33, 2], [0, 130, 7, 100, 63], hq, hkv, hd, dtype)


@pytest.mark.parametrize("hd", [16, 64, 128, 192, 256])
@pytest.mark.parametrize("kernel", ["plain", "few", "values"])
def test_attention_kernels_by_name(hd, kernel):
    """The same calls through every kernel, those "auto" would not choose among them."""
    attention_case([1, 3, 50], [70, 200, 20], 6, 2, hd, torch.bfloat16, kernel=kernel)
    attention_case([1, 3, 50], [70, 200, 20], 6, 2, hd, torch.bfloat16, kernel=kernel, window=33)
    attention_case([1, 3, 50], [70, 200, 20], 6, 2, hd, torch.float32, kernel=kernel)


@pytest.mark.parametrize("new,pos0", [([1, 1, 1], [500, 39, 40]), ([2, 2], [300, 63]), ([90, 1, 64], [0, 200, 129])])
@pytest.mark.parametrize("window", [1, 17, 64, 100])
@pytest.mark.parametrize("hd", [128, 64, 48])
def test_attention_in_a_window(new, pos0, window, hd):
    attention_case(new, pos0, 6, 2, hd, torch.bfloat16, window=window)


@pytest.mark.parametrize("hq,hkv,hd", [(28, 4, 128), (6, 1, 64), (16, 1, 128), (17, 1, 128), (64, 2, 128)])
@pytest.mark.parametrize("new", [1, 2, 3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_of_few_rows_over_long_sequences(hq, hkv, hd, new, dtype):
    attention_case([new, new, new], [5000, 4095, 2047 - new], hq, hkv, hd, dtype, seed=new)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new,pos0", [([1, 1], [600, 90]), ([40], [300])])
def test_attention_over_pages_of_unequal_scale(new, pos0, dtype):
    """Values of one page 2^40 times those of the next, keys alike: one key decides, and no weight may be lost before that."""
    attention_case(new, pos0, 4, 2, 64, dtype, spread=20, scale=1e-6)


@pytest.mark.parametrize("scale", [0.0, -0.1, 3.0])
def test_attention_scales(scale):
    attention_case([1, 20], [300, 64], 4, 2, 128, torch.bfloat16, scale=scale)


def test_attention_sees_a_nan_of_its_own_only():
    """A key that is NaN makes the rows NaN that see it; rows before it do not see it."""
    hq, hkv, hd = 4, 2, 64
    for kind in (0, 1):
        cache, scales = torch.ones(2, 2, hkv, PAGE, hd, device=DEV).to(torch.float8_e4m3fn), torch.ones(2, 2, hkv, device=DEV)
        cache.view(torch.uint8)[0, kind, 0, 50] = 0x7f
        plan = Plan([1, 1], [49, 50], [[0], [0]])                               # two sequences over one page, as a shared prefix would be
        out = torch.empty(2, hq * hd, dtype=torch.bfloat16, device=DEV)
        ops.attention_e4m3(torch.ones(2, hq, hd, dtype=torch.bfloat16, device=DEV), out, plan, 0, cache, scales, hq, hkv, hd, 0, 0.1)
        got = out.view(2, hq, hd).float().cpu()
        assert bool((got[0] == 1.0).all()) and bool(got[1, :2].isnan().all()) and bool((got[1, 2:] == 1.0).all())


@pytest.mark.parametrize("hd,window", [(64, 0), (128, 0), (48, 0), (64, 3)])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_nan_reaches_the_rows_that_see_it(hd, window, kind, dtype):
    """Several new rows of one sequence: a NaN in the key (or one value) at one of their positions, another one far back that only
    an unbounded mask sees."""
    hq, hkv, n, pos0, bad = 4, 1, 4, 70, 72
    cache, scales = torch.ones(2, 2, hkv, PAGE, hd, device=DEV).to(torch.float8_e4m3fn), torch.ones(2, 2, hkv, device=DEV)
    cache.view(torch.uint8)[1, kind, 0, bad - PAGE, 5] = 0xff
    if window:
        cache.view(torch.uint8)[1, :, 0, :67 - PAGE] = 0x7f
    plan = Plan([n], [pos0], [[0, 1]])
    out = torch.empty(n, hq * hd, dtype=dtype, device=DEV)
    ops.attention_e4m3(torch.ones(n, hq, hd, dtype=dtype, device=DEV), out, plan, 0, cache, scales, hq, hkv, hd, window, 0.1, "few")
    got = out.view(n, hq, hd).float().cpu()
    for i in range(n):
        sees = pos0 + i >= bad
        if not sees:
            assert bool((got[i] == 1.0).all()), i
        elif kind == 0:
            assert bool(got[i].isnan().all()), i
        else:
            assert bool(got[i, :, 5].isnan().all()) and int(got[i].isnan().sum()) == hq, i


@pytest.mark.parametrize("page", [16, 48, 128])
def test_pages_of_other_sizes(page):
    """The store takes any, the plain attention and the one over values of float32 rows too."""
    hq, hkv, hd, n, pos0 = 4, 2, 64, 150, 10
    g = torch.Generator().manual_seed(page)
    pages = [3, 0, 11, 5, 2, 1, 4, 7, 6, 8, 9][:-(-(n + pos0) // page)]
    oracle = plain.PlainCache(12, hkv, hd, page)
    cache = torch.zeros(12, 2, hkv, page, hd, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    scales = torch.ones(12, 2, hkv, device=DEV)
    for at, k in ((0, pos0), (pos0, n)):
        plan = Plan([k], [at], [pages])
        plan.groups[0].page_size = page
        x = rows_of(k, hq, hkv, hd, g, 0.1 if at == 0 else 1.0)
        q = torch.empty(k, hq, hd, device=DEV)
        ops.rope_store_e4m3(x.view(k, -1).to(DEV), hq, hkv, hd, 0, None, plan, 0, cache, scales, q)
        oracle.store(pages, at, torch.stack([x[:, hq:hq + hkv], x[:, hq + hkv:]], 1))
    kv = oracle.keys_values(pages, n + pos0)
    assert torch.equal(scales.cpu().double()[pages], oracle.scales[pages])
    want, size, dots = plain.attend(q.double().cpu(), kv, pos0, 0, 0.125)
    for kernel in ("plain", "values", "auto"):
        out = torch.empty(n, hq * hd, device=DEV)
        ops.attention_e4m3(q, out, plan, 0, cache, scales, hq, hkv, hd, 0, 0.125, kernel)
        far = (out.cpu().double().view(n, hq, hd) - want).abs() / plain.tolerance(want, size, dots, 0.125, hd, n + pos0, torch.float32)
        assert float(far.max()) <= 1.0, kernel
    with pytest.raises(ops.KernelError):
        ops.attention_e4m3(q, out, plan, 0, cache, scales, hq, hkv, hd, 0, 0.125, "few")


def test_attention_without_pages_gives_zeros():
    cache, scales = device_cache(3, 1, 64)
    for new in ([1, 1], [40, 40]):
        plan = Plan(new, [70, 10], [[0], [1]])                                  # the first one's list ends before its position
        n = plan.n_rows
        out = torch.full((n, 4 * 64), 5.0, dtype=torch.bfloat16, device=DEV)
        cache.zero_()
        ops.attention_e4m3(torch.ones(n, 4, 64, dtype=torch.bfloat16, device=DEV), out, plan, 0, cache, scales, 4, 1, 64, 0, 0.1)
        assert bool((out == 0).all())


def test_attention_does_not_depend_on_the_batch():
    """The same sequence alone, in a batch and on other pages: the same bits."""
    plan, q, out, cache, scales = attention_case([1, 1, 1, 1], [900, 20, 3000, 64], 12, 2, 128, torch.bfloat16)
    for i in range(4):
        first, last = (int(v) for v in plan.groups[0].page_off[i:i + 2])
        alone = Plan([1], [int(plan.seq_pos0[i])], [plan.groups[0].page_ids[first:last].tolist()])
        o = torch.empty(1, 12 * 128, dtype=torch.bfloat16, device=DEV)
        ops.attention_e4m3(q[i:i + 1].to(DEV), o, alone, 0, cache, scales, 12, 2, 128, 0, 128 ** -0.5)
        assert torch.equal(o[0], out[i])


# ------------------------------------------------------------------------------------------------ tables
def state(oracle):
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)                       # noqa: E731
    table = torch.full((len(oracle.lengths), oracle.width), -1, dtype=torch.int32)
    for s, pages in enumerate(oracle.pages):
        table[s, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
    return dict(lengths=i32(oracle.lengths), table=table.to(DEV), free=i32(oracle.free), n_free=i32([len(oracle.free)]))


def expect(oracle, t, slots, new, st):
    row0, pos0, rows, lists = oracle.tables(slots, new)
    n = len(rows)
    assert t.seq_row0.tolist() == row0 and t.seq_pos0.tolist() == pos0 and int(t.status) == 0
    got = torch.stack([t.row_seq, t.row_pos, t.row_slot], 1).cpu()
    assert got[:n].tolist() == [list(r) for r in rows]
    assert got[n:].tolist() == [[0, -1, -1]] * (t.n_rows - n)
    off = [0]
    for mine in lists:
        off.append(off[-1] + len(mine))
    assert t.page_off.tolist() == off
    assert t.page_ids[:off[-1]].tolist() == [p for mine in lists for p in mine]
    for s, mine in zip(slots, lists):
        assert st["table"][s, :len(mine)].tolist() == mine


@pytest.mark.parametrize("n,page,longest", [(1, 64, 1), (1, 64, 5000), (7, 64, 300), (33, 16, 90), (512, 64, 3), (513, 64, 70), (1500, 1, 4)])
def test_tables_through_many_steps(n, page, longest):
    rng = random.Random(n)
    n_slots, width = n + 5, 4 * (-(-longest // page)) + 1
    oracle = plain.PlainPages(n_slots, width, rng.sample(range(n_slots * width + 3), n_slots * width + 3), page)
    st = state(oracle)
    held = n_slots * width + 3
    for step in range(4):
        slots = rng.sample(range(n_slots), n)
        new = [rng.choice([0, 1, rng.randint(0, longest)]) for _ in range(n)]
        new[0] = longest
        t = ops.PageTables(n, max(1, sum(new)) + rng.choice([0, 9]), max(1, sum(-(-(oracle.lengths[s] + k) // page) for s, k in zip(slots, new))), DEV, page)
        s32, n32 = (torch.tensor(v, dtype=torch.int32, device=DEV) for v in (slots, new))
        for _ in range(2):                                                      # twice: nothing is taken before the step is recorded
            ops.page_tables(s32, n32, st["lengths"], st["table"], st["free"], st["n_free"], t, longest, width * page)
            t.check()
            expect(oracle, t, slots, new, st)
        ops.page_advance(s32, n32, st["lengths"], st["n_free"], t)
        oracle.advance(slots, new)
        assert st["lengths"].tolist() == oracle.lengths and int(st["n_free"]) == len(oracle.free)
        gone = rng.sample(range(n_slots), n_slots // 3) + [0, 0]                # one of them twice
        st_free = st["free"]
        assert st_free.numel() == held
        ops.page_release(torch.tensor(gone, dtype=torch.int32, device=DEV), st["lengths"], st["table"], st_free, st["n_free"], page)
        oracle.release(gone)
        assert st["lengths"].tolist() == oracle.lengths and st_free[:int(st["n_free"])].tolist() == oracle.free


@pytest.mark.parametrize("slots,new,kw,status", [
    ([0, 9], [1, 1], {}, 1), ([0, -1], [1, 1], {}, 1), ([2, 2], [1, 1], {}, 1), ([0, 1], [1, -1], {}, 1), ([0, 1], [1, 5], {}, 2),
    ([0, 1], [4, 4], dict(max_len=66), 2), ([3, 1], [4, 1], {}, 2), ([0, 1], [4, 4], dict(max_rows=7), 4), ([1, 3], [1, 1], dict(max_pages=3), 8),
    # 62 + 1 and 63 + 1 tokens fit a page each: two pages are enough
    ([0, 1], [1, 1], dict(max_pages=2), 0),
    # 66, 67 and 65 tokens of sequences with a page each: a new page for every one of them
    ([0, 1, 2], [4, 4, 1], dict(free=1), 16), ([0, 1, 2], [4, 4, 1], dict(free=2), 16), ([0, 1, 2], [4, 4, 1], dict(free=3), 0),
    ([0, 0], [1, 5], dict(max_rows=1), 1), ([0, 1], [0, 0], {}, 0)])
def test_tables_that_cannot_be_made_describe_no_rows(slots, new, kw, status):
    oracle = plain.PlainPages(6, 3, list(range(20, 20 + kw.get("free", 8))))
    for s, n in enumerate([62, 63, 64, 191]):
        oracle.lengths[s], oracle.pages[s] = n, [s * 3 + j for j in range(oracle.count(n))]
    st = state(oracle)
    before = {k: v.clone() for k, v in st.items()}
    t = ops.PageTables(len(slots), kw.get("max_rows", 32), kw.get("max_pages", 32), DEV)
    s32, n32 = (torch.tensor(v, dtype=torch.int32, device=DEV) for v in (slots, new))
    ops.page_tables(s32, n32, st["lengths"], st["table"], st["free"], st["n_free"], t, 4, kw.get("max_len", 192))
    assert int(t.status) == status == oracle.status(slots, new, t.n_rows, t.max_pages, 4, kw.get("max_len", 192))
    if status == 0:
        expect(oracle, t, slots, new, st)
        return
    with pytest.raises(ops.KernelError):
        t.check()
    assert t.seq_row0.tolist() == [0] * (len(slots) + 1) == t.page_off.tolist()
    assert bool((t.row_pos == -1).all()) and bool((t.row_slot == -1).all())
    ops.page_advance(s32, n32, st["lengths"], st["n_free"], t)
    assert all(torch.equal(before[k], st[k]) for k in st)
    # and the kernels behind it leave everything as it is
    cache, scales = device_cache(30, 1, 32)
    kept = cache.view(torch.uint8).clone()
    q, out = (torch.full((t.n_rows, 2, 32), 3.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    ops.rope_store_e4m3(torch.ones(t.n_rows, 4 * 32, device=DEV), 2, 1, 32, 0, None, t, 0, cache, scales, q)
    ops.attention_e4m3(q, out, t, 0, cache, scales, 2, 1, 32, 0, 0.1)
    assert bool((q == 3.0).all()) and bool((out == 3.0).all()) and torch.equal(kept, cache.view(torch.uint8))


# ------------------------------------------------------------------------------------------------ together
def test_all_of_them_in_a_replayed_graph():
    """Prompts eagerly, then a captured step (tables, store, attention, advance) replayed token by token across page ends, with the
    host giving nothing but new rows: against the plain form, token by token."""
    hq, hkv, hd, n = 6, 2, 64, 5
    g = torch.Generator().manual_seed(3)
    oracle_pages = plain.PlainPages(n + 2, 4, list(range(40)))
    st = state(oracle_pages)
    oracle = plain.PlainCache(40, hkv, hd)
    cache, scales = device_cache(40, hkv, hd)
    slots, scale, rot = [3, 0, 6, 2, 5], hd ** -0.5, 64
    inv = torch.exp(torch.arange(0, rot, 2) * (-math.log(1e4) / rot)).to(DEV)
    s32 = torch.tensor(slots, dtype=torch.int32, device=DEV)

    def one_step(t, n32, x, q, out):
        ops.page_tables(s32, n32, st["lengths"], st["table"], st["free"], st["n_free"], t, t.n_rows, 256)
        angles = ops.rotation_table(t.row_pos, inv, rot)
        ops.rope_store_e4m3(x, hq, hkv, hd, rot, angles, t, 0, cache, scales, q)
        ops.attention_e4m3(q, out, t, 0, cache, scales, hq, hkv, hd, 0, scale)
        ops.page_advance(s32, n32, st["lengths"], st["n_free"], t)
        return angles

    def check(new, x, angles, out):
        row0, pos0, _, lists = oracle_pages.tables(slots, new)
        host, cs = x.cpu().view(-1, hq + 2 * hkv, hd), angles.cpu()
        for i, k in enumerate(new):
            if not k:
                continue
            rows = host[row0[i]:row0[i + 1]].clone()
            c = cs[row0[i]:row0[i + 1], None]
            rows[:, :hq + hkv] = plain.rotate(rows[:, :hq + hkv], c[..., :rot // 2], c[..., rot // 2:])
            oracle.store(lists[i], pos0[i], torch.stack([rows[:, hq:hq + hkv], rows[:, hq + hkv:]], 1))
            want, size, dots = plain.attend(rows[:, :hq].to(torch.bfloat16).double(), oracle.keys_values(lists[i], pos0[i] + k), pos0[i], 0, scale)
            got = out[row0[i]:row0[i + 1]].cpu().double().view(k, hq, hd)
            assert float(((got - want).abs() / plain.tolerance(want, size, dots, scale, hd, pos0[i] + k, torch.bfloat16)).max()) <= 1.0
        oracle_pages.advance(slots, new)
        assert st["lengths"].tolist() == oracle_pages.lengths and int(st["n_free"]) == len(oracle_pages.free)

    def buffers(rows):
        return (torch.empty(rows, (hq + 2 * hkv) * hd, device=DEV), torch.empty(rows, hq, hd, dtype=torch.bfloat16, device=DEV),
                torch.empty(rows, hq * hd, dtype=torch.bfloat16, device=DEV))

    new = [30, 64, 1, 100, 126]
    x, q, out = buffers(sum(new))
    x.copy_(torch.randn(x.shape, generator=g))
    t = ops.PageTables(n, sum(new), 20, DEV)
    n32 = torch.tensor(new, dtype=torch.int32, device=DEV)
    check(new, x, one_step(t, n32, x, q, out), out)

    new = [1, 1, 0, 1, 1]                                                       # one of them sits out: its row is a spare one
    x, q, out = buffers(n)
    t = ops.PageTables(n, n, 20, DEV)
    n32 = torch.tensor(new, dtype=torch.int32, device=DEV)
    before = {k: v.clone() for k, v in st.items()}
    saved = cache.view(torch.uint8).clone(), scales.clone()
    x.zero_()
    one_step(t, n32, x, q, out)                                                 # set-up run: put back what it changed
    torch.cuda.synchronize()
    for k, v in before.items():
        st[k].copy_(v)
    cache.view(torch.uint8).copy_(saved[0]), scales.copy_(saved[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        angles = one_step(t, n32, x, q, out)
    for _ in range(70):
        x.copy_(torch.randn(x.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        t.check()
        check(new, x, angles, out)


def test_on_another_stream():
    """Work of a side stream: ordered there, the same bits as on the default stream."""
    plan, q, out, cache, scales = attention_case([1, 1, 40], [900, 20, 64], 12, 2, 128, torch.bfloat16)
    side, other = torch.cuda.Stream(), torch.full_like(out, 5.0)
    q = q.to(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.attention_e4m3(q, other, plan, 0, cache, scales, 12, 2, 128, 0, 128 ** -0.5)
    side.synchronize()
    assert torch.equal(out, other)


def test_refusals_in_python():
    cache, scales = device_cache(3, 1, 64)
    plan = Plan([1], [3], [[0]])
    q, out = (torch.zeros(1, 2, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    qkv = torch.zeros(1, 4 * 64, device=DEV)
    good = (q, out, plan, 0, cache, scales, 2, 1, 64, 0, 0.1)
    ops.attention_e4m3(*good)
    with pytest.raises(ops.KernelError):
        ops.attention_e4m3(q, q, *good[2:])
    for i, bad in [(4, cache.float()), (4, cache[:, :, :, :32]), (5, scales.double()), (5, scales[:2]), (0, q.float()), (0, q[:, :1]), (6, 3), (8, 32)]:
        args = list(good)
        args[i] = bad
        with pytest.raises((AssertionError, ops.KernelError)):
            ops.attention_e4m3(*args)
    good = (qkv, 2, 1, 64, 0, None, plan, 0, cache, scales, q)
    ops.rope_store_e4m3(*good)
    for i, bad in [(0, qkv.bfloat16()), (0, qkv[:, :64]), (4, 64), (4, 3), (5, torch.zeros(1, 6, device=DEV)), (8, cache.view(torch.uint8)), (9, scales[:, :1]),
                   (10, q.half()), (10, q[:, :1])]:
        args = list(good)
        args[i] = bad
        with pytest.raises((AssertionError, ops.KernelError)):
            ops.rope_store_e4m3(*args)


@pytest.mark.parametrize("hd,later", [(64, 1), (64, 20), (22, 1)])
def test_store_goes_from_the_smallest_to_the_largest_scale(hd, later):
    """Numbers of a page whose scale grows beyond their whole range become zeros; one whose scale grows by less keeps them."""
    cache, scales = device_cache(1, 1, hd)
    q = torch.empty(30, 1, hd, device=DEV)
    at = 0
    for n, size, exponent, first in ((3, 2.0 ** -118, -126, 256.0), (later, 2.0 ** -110, -118, 1.0), (2, 2.0 ** 100, 92, 0.0)):
        ops.rope_store_e4m3(torch.full((n, 3 * hd), size, device=DEV), 1, 1, hd, 0, None, Plan([n], [at], [[0]]), 0, cache, scales, q[:n])
        at += n
        # size / 2^exponent is 256, within 448 and above 224; the first token's numbers 256 * 2^(-126 - exponent)
        assert scales.flatten().tolist() == [2.0 ** exponent] * 2
        assert bool((cache.float()[0, :, 0, at - n:at] == 256.0).all()) and bool((cache.float()[0, :, 0, :3] == (256.0 if at == 3 else first)).all())


def test_release_of_lengths_that_no_table_holds():
    """Lengths up to the largest int: a slot gives back as many pages as its table has, the stack keeps to its room."""
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)                       # noqa: E731
    lengths, table, free, n_free = i32([2 ** 31 - 1, 65, -5]), i32([[5, 6], [7, 8], [9, 10]]), i32([0, 1, -1, -1, -1]), i32([2])
    ops.page_release(i32([0, 2, 1]), lengths, table, free, n_free)
    # three places are left: slot 0's two pages, slot 2 has none, slot 1's first
    assert free.tolist() == [0, 1, 5, 6, 7] and int(n_free) == 5
    assert lengths.tolist() == [0, 0, 0] and table.tolist() == [[-1, -1], [-1, -1], [9, 10]]
    n_free.fill_(-7)
    lengths.copy_(i32([1, 0, 0]))
    table[0, 0] = 3
    ops.page_release(i32([0]), lengths, table, free, n_free)
    assert free.tolist() == [3, 1, 5, 6, 7] and int(n_free) == 1


def test_tables_of_lengths_that_no_table_holds():
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)                       # noqa: E731
    t = ops.PageTables(2, 8, 8, DEV)
    for held in (2 ** 31 - 1, 2 ** 31 - 64, -1):
        ops.page_tables(i32([0, 1]), i32([1, 1]), i32([held, 3]), i32([[0, 1], [2, 3]]), i32([4]), i32([1]), t, 1, 2 ** 31 - 1)
        assert int(t.status) == 2 and t.seq_row0.tolist() == [0, 0, 0] and bool((t.row_slot == -1).all())


def test_rows_that_share_memory_are_refused():
    cache, scales = device_cache(3, 1, 64)
    plan = Plan([1], [3], [[0]])
    memory = torch.zeros(512, device=DEV)
    with pytest.raises(ops.KernelError, match="share memory"):
        ops.rope_store_e4m3(memory[:256].view(1, 256), 2, 1, 64, 0, None, plan, 0, cache, scales, memory[128:256].view(1, 2, 64))
    ops.rope_store_e4m3(memory[:256].view(1, 256), 2, 1, 64, 0, None, plan, 0, cache, scales, memory[256:384].view(1, 2, 64))
    with pytest.raises(ops.KernelError, match="share memory"):
        ops.attention_e4m3(memory[:128].view(1, 2, 64), memory[64:192].view(1, 2, 64), plan, 0, cache, scales, 2, 1, 64, 0, 0.1)
    ops.attention_e4m3(memory[:128].view(1, 2, 64), memory[128:256].view(1, 2, 64), plan, 0, cache, scales, 2, 1, 64, 0, 0.1)


def test_room_for_values_goes_by_the_step_and_not_by_the_pool():
    """A prompt's attention by way of values takes room for the pages that its requests can have, not for all there are."""
    pages = DevicePages(4, 4096, 1024, DEV)
    tables = pages.tables(2, 300)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)                       # noqa: E731
    slots, new = i32([3, 1]), i32([200, 70])
    pages.plan(slots, new, tables, 200, 256)
    cache, scales = device_cache(16, 1, 64)
    g = torch.Generator().manual_seed(9)
    qkv = torch.randn(300, 4 * 64, generator=g).to(DEV)
    q, few, values = (torch.zeros(300, 2, 64, dtype=torch.bfloat16, device=DEV) for _ in range(3))
    ops.rope_store_e4m3(qkv, 2, 1, 64, 0, None, tables, 0, cache, scales, q)
    ops.attention_e4m3(q, few, tables, 0, cache, scales, 2, 1, 64, 0, 0.125, kernel="few")
    ops.attention_e4m3(q, values, tables, 0, cache, scales, 2, 1, 64, 0, 0.125, kernel="values")
    # 8 pages of 2 * 64 * 64 values in bfloat16, their numbers, partial rows of 4 splits of 300 * 2 rows at most: under 2 MB
    assert tables.groups[0].page_ids.numel() == 8 and sum(t.numel() for t in tables._scratch) < 2 << 20
    # values of size 1, weights that add up to 1: the two differ by roundings of the weights (2^-8) and of the results (2^-8), times |v| < 8
    assert float((few[:270].float() - values[:270].float()).abs().max()) <= 8 * 2.0 ** -7 and bool((values[270:] == 0).all())
    # a longer bound gives the whole room back
    pages.plan(slots, new, tables, 200)
    assert tables.groups[0].page_ids.numel() == 2048
