"""The 8-bit cache on a machine without a GPU: the plain form against torch's own e4m3, and what the entry points refuse before
anything is launched (no address given here is one of a device: a call that is not refused would not come back with these codes)."""
import math
import re
from pathlib import Path

import pytest
import torch

import plain_cache_e4m3 as plain
from sonicboom_b200 import abi, ops

ARG, UNSUPPORTED = 1, 2
P = 4096                                                  # an address that nothing reads


def test_rounding_is_torchs():
    x = torch.randn(20000, dtype=torch.float64) * torch.exp2(torch.randint(-14, 7, (20000,)).double())
    x = torch.cat([x.clamp(-448, 448), torch.tensor([0.0, 2.0 ** -10, 3 * 2.0 ** -10, 448.0, -448.0, 17.0, 19.0], dtype=torch.float64)])
    x = x.float()
    assert torch.equal(plain.round_e4m3(x.double()), x.to(torch.float8_e4m3fn).double())
    assert plain.round_e4m3(torch.tensor([math.inf, -math.inf, math.nan], dtype=torch.float64)).isnan().all()


@pytest.mark.parametrize("largest,e", [(448.0, 0), (math.nextafter(448.0, 1e9), 1), (224.0, -1), (1.0, -8), (0.0, -126), (1e-40, -126),
                                       (3.4028234663852886e38, 120)])
def test_exponents(largest, e):
    assert plain.exponent_for(largest) == e


def test_a_larger_scale_rounds_only_what_is_not_normal_any_more():
    c = plain.PlainCache(1, 1, 16)
    first = 1.7 * torch.exp2(-torch.arange(96).float() / 6).view(3, 2, 1, 16)     # down to 2^-15: around the new scale's 2^-9
    first[0, :, 0, 0] = 3.0
    c.store([0], 0, first)
    before = c.keys_values([0], 3)
    c.store([0], 3, torch.full((1, 2, 1, 16), 50.0))      # 16 to 17 times the largest: four or five steps of the exponent
    after = c.keys_values([0], 4)[:, :, :3]
    scale = float(c.scales[0, 0, 0])
    normal = before.abs() >= 2.0 ** -6 * scale
    assert torch.equal(before[normal], after[normal]) and bool(normal.any()) and bool((~normal).any())
    assert float((before - after).abs().max()) <= 2.0 ** -10 * scale


def record(name, *values):
    return abi.pack[name](*(0 if v is None else v for v in values))


def test_records_are_the_headers_structs():
    text = re.sub(r"/\*.*?\*/", " ", (Path(abi.__file__).parent / "csrc" / "sonicboom_b200.h").read_text(), flags=re.S)
    for name, codes in abi.RECORDS.items():
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
        found = ""
        for decl in filter(None, (d.strip() for d in body.split(";"))):
            code = "p" if "*" in decl else {"int": "i", "float": "f", "size_t": "z"}[decl.split()[0]]
            found += code * (decl.count(",") + 1)
        assert found == codes, name
    for name in ("sb_rope_store_e4m3", "sb_page_tables"):
        assert getattr(ops.lib(), name)(None, None) == ARG


def store(l, qkv=P, rows=4, seqs=2, max_new=2, hq=4, hkv=2, hd=64, rot=64, angles=P, row0=P, pos0=P, off=P, ids=P, page=64, cache=P,
          scales=P, pages=8, q=P, dtype=1):
    return l.sb_rope_store_e4m3(record("SbStoreE4m3", qkv, angles, row0, pos0, off, ids, cache, scales, q, rows, seqs, max_new, hq, hkv, hd,
                                       rot, page, pages, dtype, 148), None)


@pytest.mark.parametrize("kw,code", [
    (dict(qkv=None), ARG), (dict(cache=None), ARG), (dict(scales=None), ARG), (dict(q=None), ARG), (dict(ids=None), ARG),
    (dict(rows=0), ARG), (dict(seqs=0), ARG), (dict(max_new=0), ARG), (dict(hq=0), ARG), (dict(hkv=0), ARG), (dict(page=0), ARG),
    (dict(pages=0), ARG), (dict(hd=63), ARG), (dict(rot=66), ARG), (dict(rot=31), ARG), (dict(rot=-2), ARG), (dict(angles=None), ARG),
    (dict(dtype=7), ARG), (dict(seqs=65536), UNSUPPORTED), (dict(hq=65535), UNSUPPORTED)])
def test_store_refusals(kw, code):
    l = ops.lib()
    assert store(l, **kw) == code and b"sb_rope_store_e4m3" in l.sb_last_error()


def attend(l, q=P, out=P, dtype=1, rows=4, seq=P, pos=P, off=P, ids=P, page=64, cache=P, scales=P, pages=8, hq=4, hkv=2, hd=64, window=0):
    return l.sb_attention_e4m3_plain(q, out, dtype, rows, seq, pos, off, ids, page, cache, scales, pages, hq, hkv, hd, window, 0.125, None)


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), ARG), (dict(cache=None), ARG), (dict(scales=None), ARG), (dict(rows=0), ARG), (dict(page=0), ARG), (dict(pages=0), ARG),
    (dict(hq=5), ARG), (dict(window=-1), ARG), (dict(dtype=2), ARG), (dict(hd=1026), UNSUPPORTED), (dict(hq=65536), UNSUPPORTED)])
def test_plain_attention_refusals(kw, code):
    l = ops.lib()
    assert attend(l, **kw) == code and b"sb_attention_e4m3_plain" in l.sb_last_error()


def values(l, row0=P, pos0=P, seqs=2, max_len=100, off=P, ids=P, n_list=4, page=64, cache=P, scales=P, pages=8, hq=4, hkv=2, hd=64, window=0,
           out=P, dtype=1, numbers=P, rows=P):
    return l.sb_cache_e4m3_values(row0, pos0, seqs, max_len, off, ids, n_list, page, cache, scales, pages, hq, hkv, hd, window, out, dtype,
                                  numbers, rows, None)


@pytest.mark.parametrize("kw,code", [
    (dict(row0=None), ARG), (dict(cache=None), ARG), (dict(out=None), ARG), (dict(numbers=None), ARG), (dict(rows=None), ARG),
    (dict(seqs=0), ARG), (dict(max_len=0), ARG), (dict(n_list=0), ARG), (dict(page=0), ARG), (dict(pages=0), ARG), (dict(window=-1), ARG),
    (dict(hd=66), UNSUPPORTED), (dict(out=P + 8), UNSUPPORTED), (dict(dtype=3), ARG), (dict(seqs=65536), UNSUPPORTED)])
def test_values_refusals(kw, code):
    l = ops.lib()
    assert values(l, **kw) == code and b"sb_cache_e4m3_values" in l.sb_last_error()


def tables(l, slots=P, new=P, n=4, lengths=P, table=P, n_slots=8, width=4, free=P, pages=32, n_free=P, page=64, max_rows=16, max_pages=16,
           max_new=4, max_len=256, outs=(P,) * 8):
    return l.sb_page_tables(record("SbPageTables", slots, new, lengths, table, free, n_free, *outs, n, n_slots, width, pages, page, max_rows,
                                   max_pages, max_new, max_len), None)


@pytest.mark.parametrize("kw,code", [
    (dict(slots=None), ARG), (dict(new=None), ARG), (dict(lengths=None), ARG), (dict(table=None), ARG), (dict(free=None), ARG),
    (dict(n_free=None), ARG), (dict(outs=(P,) * 7 + (None,)), ARG), (dict(n=0), ARG), (dict(n_slots=0), ARG), (dict(width=0), ARG),
    (dict(pages=0), ARG), (dict(page=0), ARG), (dict(max_rows=0), ARG), (dict(max_pages=0), ARG), (dict(max_new=0), ARG),
    (dict(max_len=0), ARG), (dict(n=8193), UNSUPPORTED), (dict(n_slots=(1 << 18) + 1), UNSUPPORTED), (dict(max_rows=(1 << 21) + 1), UNSUPPORTED),
    (dict(width=(1 << 21) + 1), UNSUPPORTED), (dict(pages=1 << 26), UNSUPPORTED)])
def test_tables_refusals(kw, code):
    l = ops.lib()
    assert tables(l, **kw) == code and b"sb_page_tables" in l.sb_last_error()


def test_advance_and_release_refusals():
    l = ops.lib()
    assert l.sb_page_advance(None, P, 2, P, 4, P, 64, P, None) == ARG
    assert l.sb_page_advance(P, P, 2, P, 4, P, 64, None, None) == ARG
    assert l.sb_page_advance(P, P, 0, P, 4, P, 64, P, None) == ARG
    assert l.sb_page_release(P, 2, P, None, 4, 8, P, 8, P, 64, None) == ARG
    assert l.sb_page_release(P, 2, P, P, 4, 0, P, 8, P, 64, None) == ARG
    assert l.sb_page_release(P, 8193, P, P, 4, 8, P, 8, P, 64, None) == UNSUPPORTED


def test_tensors_that_are_not_on_a_gpu_are_refused():
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ops.KernelError):
        ops.page_tables(i, i, i, torch.zeros(2, 4, dtype=torch.int32), i, i[:1], ops.PageTables(2, 4, 4, "cpu"), 1, 64)


# ------------------------------------------------------------------------------------------------ cache and engine
def test_cache_storage_and_scales():
    from sonicboom_b200.cache import Cache, KVNeed
    from sonicboom_b200.cache.kv import E4M3
    c = Cache([KVNeed(2, 32), None, KVNeed(2, 32), KVNeed(1, 16, 40)], [None] * 4, 640, torch.bfloat16, "cpu", kv_dtype=E4M3)
    assert [g.storage.dtype for g in c.groups] == [E4M3, E4M3]
    assert c.groups[0].entry_storage(2).shape == (10, 2, 2, 64, 32) and c.groups[0].entry_scales(2).shape == (10, 2, 2)
    assert c.groups[0].scales.dtype == torch.float32 and c.groups[0].bytes_per_token() == 2 * 2 * 2 * 32
    plain_cache = Cache([KVNeed(2, 32)], [None], 640, torch.bfloat16, "cpu")
    assert plain_cache.groups[0].scales is None and plain_cache.groups[0].entry_scales(0) is None
    assert plain_cache.groups[0].storage.dtype == torch.bfloat16


def test_engine_takes_it_for_plain_attention_only():
    from conftest import TINY
    from sonicboom_b200 import DecoderModel, Engine
    from sonicboom_b200.cache.kv import E4M3
    from sonicboom_b200.config import spec_from_config_dict
    model = DecoderModel(spec_from_config_dict(TINY["C"])[1], torch.bfloat16, "cpu")
    assert all(g.storage.dtype == E4M3 for g in Engine(model, 256, cache_dtype="e4m3").cache.groups)
    assert all(g.storage.dtype == torch.bfloat16 for g in Engine(model, 256).cache.groups)
    with pytest.raises(ValueError, match="cache_dtype"):
        Engine(model, 256, cache_dtype="int8")
    import zolulix_util
    other = DecoderModel(spec_from_config_dict(next(iter(zolulix_util.CONFIGS.values())))[1], torch.bfloat16, "cpu")
    with pytest.raises(ValueError, match="does not take"):
        Engine(other, 256, cache_dtype="e4m3")


def test_device_pages_refuse_sizes_without_room():
    from sonicboom_b200.cache import CacheError, DevicePages
    for sizes in ((0, 4, 4), (4, 0, 4), (4, 4, 0)):
        with pytest.raises(CacheError):
            DevicePages(*sizes, "cpu")


def test_which_rows_attend_to_pages_as_they_are():
    """A rule on sizes that needs no device: single tokens always, many bfloat16 rows by way of values, float32 rows as far as the
    grid goes."""
    class Plan:
        def __init__(self, n_seqs, max_new, max_len):
            self.n_seqs, self.max_new, self.max_len, self.n_rows = n_seqs, max_new, max_len, n_seqs * max_new

    def direct(dtype, *plan):
        return ops._reads_pages_directly(Plan(*plan), dtype, 28, 4, 128, 148)

    bf16, f32 = torch.bfloat16, torch.float32
    assert direct(bf16, 64, 1, 32768) and direct(bf16, 1, 2, 1 << 20) and direct(bf16, 1, 16, 16000) and direct(bf16, 8, 9, 4000)
    assert not direct(bf16, 1, 2048, 2048) and not direct(bf16, 8, 64, 4000)
    assert direct(f32, 1, 2048, 2048) and not direct(f32, 1, 65536, 65536) and not direct(f32, 1, 32768, 32768)


def attend_direct(l, q=P, out=2 * P, dtype=1, rows=4, seqs=2, max_new=2, max_len=100, row0=P, pos0=P, off=P, ids=P, page=64, cache=P, scales=P,
                  pages=8, hq=4, hkv=2, hd=64, window=0, scratch=P, room=1 << 20):
    return l.sb_attention_e4m3(record("SbAttentionE4m3", q, out, row0, pos0, off, ids, cache, scales, scratch, room, dtype, rows, seqs, max_new,
                                      max_len, page, pages, hq, hkv, hd, window, 0.125), None)


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), ARG), (dict(out=None), ARG), (dict(cache=None), ARG), (dict(scales=None), ARG), (dict(ids=None), ARG), (dict(rows=0), ARG),
    (dict(seqs=0), ARG), (dict(max_new=0), ARG), (dict(max_len=0), ARG), (dict(pages=0), ARG), (dict(hq=5), ARG), (dict(window=-1), ARG),
    (dict(dtype=2), ARG), (dict(hd=128), ARG), (dict(q=P + 8), ARG), (dict(scratch=P + 8), ARG), (dict(page=32), UNSUPPORTED),
    (dict(seqs=65536), UNSUPPORTED), (dict(max_new=65536), UNSUPPORTED), (dict(max_len=2000, room=100), ARG),
    (dict(max_len=2000, scratch=None), ARG), (dict(max_len=2 ** 31 - 1), UNSUPPORTED)])
def test_attention_refusals(kw, code):
    l = ops.attention_lib(64)
    assert attend_direct(l, **kw) == code and b"sb_attention_e4m3" in l.sb_last_error()
    assert l.sb_attention_e4m3(None, None) == ARG
