"""The 8-bit cache's entry points at the limits of what they take, on a machine without a GPU."""
import ctypes

import pytest
import torch

from sonicboom_b200 import abi, ops


@pytest.mark.parametrize("name", list(abi.RECORDS))
def test_a_packed_record_is_as_long_as_its_struct(name):
    """An entry point copies the whole struct, the padding behind its last member too."""
    of = {"p": ctypes.c_void_p, "z": ctypes.c_size_t, "i": ctypes.c_int, "f": ctypes.c_float}
    struct = type(name, (ctypes.Structure,), {"_fields_": [(f"m{i}", of[c]) for i, c in enumerate(abi.RECORDS[name])]})
    assert len(abi.pack[name](*[0] * len(abi.RECORDS[name]))) == abi.RECORD_STRUCTS[name].size == ctypes.sizeof(struct)


# ------------------------------------------------------------------------------------------------ calls that a fake library records
class Recorder:
    """A library whose entry points note their arguments and succeed."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def entry(*args):
            self.calls.append((name, args))
            return 0
        return entry


@pytest.fixture
def recorder(monkeypatch):
    """The operators on host tensors, as far as their calls of the library: nothing is computed."""
    r = Recorder()
    monkeypatch.setattr(ops, "_device_of", lambda t, what: -1)
    monkeypatch.setattr(ops, "_stream_of", lambda index: 0)
    monkeypatch.setattr(ops, "_sm_count", lambda index: 148)
    monkeypatch.setattr(ops, "lib", lambda: r)
    monkeypatch.setattr(ops, "attention_lib", lambda head_dim: r)
    monkeypatch.setattr(ops, "_attn_counters", lambda n, device: torch.zeros(n, dtype=torch.int32))
    return r


def i32(values):
    return torch.tensor(values, dtype=torch.int32)


class Plan:
    def __init__(self, new, pos0, lists):
        self.n_seqs, self.n_rows, self.max_new, self.max_len = len(new), sum(new), max(new), max(p + n for p, n in zip(pos0, new))
        row0, off = [0], [0]
        for n, pages in zip(new, lists):
            row0.append(row0[-1] + n)
            off.append(off[-1] + len(pages))
        self.seq_row0, self.seq_pos0 = i32(row0), i32(pos0)
        self.row_seq = i32([i for i, n in enumerate(new) for _ in range(n)])
        self.row_pos = i32([p + j for p, n in zip(pos0, new) for j in range(n)])
        self.groups = [ops.TableGroup(i32(off), i32([p for pages in lists for p in pages]), 64)]

    def scratch(self, nbytes, device):
        return torch.empty(nbytes, dtype=torch.uint8) if nbytes else None


def attend(plan, hq=4, hkv=2, hd=64, dtype=torch.bfloat16, kernel="auto", window=0):
    cache = torch.zeros(4, 2, hkv, 64, hd, dtype=torch.uint8).view(torch.float8_e4m3fn)
    q, out = (torch.zeros(plan.n_rows, hq, hd, dtype=dtype) for _ in range(2))
    return ops.attention_e4m3(q, out, plan, 0, cache, torch.ones(4, 2, hkv), hq, hkv, hd, window, 0.125, kernel)


@pytest.mark.parametrize("field", ["row_seq", "row_pos"])
def test_the_plain_kernels_row_arrays_are_checked(recorder, field):
    """It reads a sequence and a position for every row."""
    plan = Plan([1, 2], [70, 5], [[0, 1], [2]])
    attend(plan, kernel="plain")
    assert [name for name, _ in recorder.calls] == ["sb_attention_e4m3_plain"]
    good = getattr(plan, field)
    for bad in (good[:2], good.long(), torch.stack([good, good])):
        setattr(plan, field, bad)
        with pytest.raises(ops.KernelError, match="attention_e4m3"):
            attend(plan, kernel="plain")
    assert len(recorder.calls) == 1


@pytest.mark.parametrize("hq,hkv,new", [(4, 2, [1, 1]), (28, 4, [2]), (16, 1, [1]), (17, 1, [1]), (4, 2, [40, 3])])
def test_values_are_read_by_kernels_that_wait_for_them(recorder, hq, hkv, new):
    """The kernels of `attention` for few rows read old pages ahead of their wait for the kernel before them; here that one has
    just written them.  So the call asks for more rows a key/value head than those kernels take."""
    plan = Plan(new, [70] * len(new), [[0, 1], [2, 3]][:len(new)])
    attend(plan, hq, hkv, kernel="values")
    (args,) = [args for name, args in recorder.calls if name == "sb_attention"]
    assert args[4] >= plan.max_new and args[4] * (hq // hkv) > ops.DECODE_ATTENTION_ROWS


# ------------------------------------------------------------------------------------------------ tokens that are taken back
def test_a_cache_in_8_bits_goes_back_to_whole_pages():
    """What is left of a page's numbers goes back to all tokens that were written to it, the cut ones too."""
    from sonicboom_b200.cache import Cache, KVNeed
    from sonicboom_b200.cache.kv import E4M3

    def cut(kv_dtype, *lengths, window=0, held=300):
        c = Cache([KVNeed(1, 16), KVNeed(1, 16, window)], [None] * 2, 640, torch.bfloat16, "cpu", kv_dtype=kv_dtype)
        slot = c.open()
        c.reserve(slot, held)
        c.advance(slot, held)
        done = [c.truncate(slot, n) for n in lengths]
        c.check()
        return done, c.length(slot), len(c.page_list(slot, 0))

    assert cut(E4M3, 300) == ([True], 300, 5)                    # nothing is cut
    assert cut(E4M3, 299) == ([True], 256, 4) and cut(E4M3, 256) == ([True], 256, 4)
    assert cut(E4M3, 299, 256, 200, 63) == ([True] * 4, 0, 0)
    assert cut(None, 299) == ([True], 299, 5) and cut(None, 63) == ([True], 63, 1)
    # a window of 40 at 300 tokens has given the pages before 261 back: 299 goes back to 256, whose next token reads 217
    assert cut(E4M3, 299, window=40) == ([False], 300, 5)
    assert cut(E4M3, 300, window=40) == ([True], 300, 5) and cut(None, 299, window=40) == ([True], 299, 5)


def test_scratch_memory_of_tables_that_grow_step_by_step():
    """Every buffer stays for the graphs that know it; together they are bounded by what is needed."""
    t = ops.PageTables(1, 4, 4, "cpu")
    first = t.scratch(100, "cpu")
    for n in range(100, 20000, 7):
        got = t.scratch(n, "cpu")
        assert got.numel() >= n and sum(b.numel() for b in t._scratch) < 4 * n
        assert t.scratch(n // 2, "cpu") is got
    assert t._scratch[0] is first and t.scratch(0, "cpu") is None and len(t._scratch) <= 9


# ------------------------------------------------------------------------------------------------ plans made on the device
def make_tables(n=2, tables=None):
    tables = tables or ops.PageTables(n, 4, 8, "cpu")
    one = torch.ones(n, dtype=torch.int32)
    return ops.page_tables(i32(list(range(n))), one, one, torch.zeros(n, 4, dtype=torch.int32), i32([0] * 8), i32([8]), tables, 1, 256)


def test_kernels_that_read_a_plan_early_are_kept_apart_from_the_one_that_makes_it(recorder, monkeypatch):
    """Once for every making of the tables, ahead of the first kernel that may read one of their arrays before its wait; not for
    kernels that wait first."""
    monkeypatch.setattr(ops, "_ptr", lambda t: None if t is None else t.data_ptr())
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    names = lambda: [name for name, _ in recorder.calls if not name.endswith("_bytes")]                      # noqa: E731
    q, out = (torch.zeros(4, 4, 22, dtype=torch.bfloat16) for _ in range(2))

    def store(t):
        g = t.groups[0]
        ops.rope_store(torch.zeros(4, 8 * 22), 4, 2, 22, 0, torch.ones(11), t.row_seq, t.row_pos, g.page_off, g.page_ids, 64,
                       torch.zeros(8, 2, 2, 64, 22, dtype=torch.bfloat16), q)

    t, other = make_tables(), make_tables()
    ops.rotation_table(t.row_pos, torch.ones(8), 16)
    attend(t, kernel="plain")
    ops.page_advance(i32([0, 1]), i32([1, 1]), i32([1, 1]), i32([8]), t)
    assert "sb_page_tables_settle" not in names() and len(names()) == 5
    recorder.calls.clear()
    store(t)
    store(t)
    assert names() == ["sb_page_tables_settle", "sb_rope_store", "sb_rope_store"]
    recorder.calls.clear()
    ops.attention(q, out, other, 0, torch.zeros(8, 2, 2, 64, 22), 4, 2, 22, 0, 0.1, kernel="plain")
    assert names() == ["sb_page_tables_settle", "sb_attention_plain"]
    recorder.calls.clear()
    make_tables(tables=t)
    store(t)
    del t, other
    make_tables()                                                               # gone before anything reads them
    ops.rotation_table(i32([0]), torch.ones(8), 16)
    assert names() == ["sb_page_tables", "sb_page_tables_settle", "sb_rope_store", "sb_page_tables", "sb_rotation_table"]


def test_numbers_that_no_record_holds_are_refused(recorder):
    """Beyond 32 bits, or no whole numbers: the module's own error, and nothing is launched."""
    tables = ops.PageTables(2, 4, 8, "cpu")
    one, state = i32([1, 1]), (i32([0, 0]), torch.zeros(2, 4, dtype=torch.int32), i32([0] * 8), i32([8]))
    for max_new, max_len in ((2 ** 31, 256), (1, 2 ** 31), (1, 2.5)):
        with pytest.raises(ops.KernelError, match="SbPageTables"):
            ops.page_tables(i32([0, 1]), one, *state, tables, max_new, max_len)
    plan = Plan([1], [5], [[0]])
    for window in (2 ** 31, 0.5):
        with pytest.raises(ops.KernelError, match="SbAttentionE4m3"):
            attend(plan, window=window)
    plan.max_new = 2 ** 31
    cache = torch.zeros(4, 2, 2, 64, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    with pytest.raises(ops.KernelError, match="SbStoreE4m3"):
        ops.rope_store_e4m3(torch.zeros(1, 8 * 64), 4, 2, 64, 0, None, plan, 0, cache, torch.ones(4, 2, 2), torch.zeros(1, 4, 64))
    assert not [name for name, _ in recorder.calls if not name.endswith("_bytes")]


def test_device_pages_take_tables_of_their_own_page_size_only(recorder):
    """Lengths, page lists and the stack count pages of one size."""
    from sonicboom_b200.cache import CacheError, DevicePages
    pages = DevicePages(4, 8, 4, "cpu", page_size=32)
    slots, one = i32([0, 1]), i32([1, 1])
    mine = pages.tables(2, 4)
    assert mine.page_size == 32 and mine.max_pages == 8 and pages.tables(2, 4, 3).max_pages == 3
    pages.plan(slots, one, mine, 1)
    pages.advance(slots, one, mine)
    other = ops.PageTables(2, 4, 8, "cpu")
    for call in (lambda: pages.plan(slots, one, other, 1), lambda: pages.advance(slots, one, other)):
        with pytest.raises(CacheError, match="tokens"):
            call()
    assert [name for name, _ in recorder.calls] == ["sb_page_tables", "sb_page_advance"]
    with pytest.raises(ops.KernelError, match="room"):
        pages.tables(2, 4, 0)
    for sizes in ((0, 4, 4), (2, 0, 4), (2, 4, -1), (2, 4, 4, "cpu", 0)):
        with pytest.raises(ops.KernelError, match="room"):
            ops.PageTables(*sizes[:3], "cpu", *sizes[4:])


def test_tables_that_are_gone_are_forgotten(recorder):
    for _ in range(50):
        make_tables()
    kept = make_tables()
    assert len(ops._unsettled) == 1 and ops._unsettled_from == kept.start and ops._unsettled_to == kept.end
