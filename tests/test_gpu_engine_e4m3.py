"""Whole models over a cache held in 8 bits: logits against the plain model whose keys and values are rounded the same way, the
same tokens in several cuts, the captured decode loop, prefix reuse, the entry points, page lists on the device."""
import pytest
import torch

import plain_cache_e4m3 as plain
import plain_model as pm
from conftest import BF16_TOLS, TINY, prompts_for
from gpu_util import _load, batch_unequal, tail_one_by_one, whole

import sonicboom_b200 as sb
from sonicboom_b200 import llm

pytestmark = pytest.mark.gpu
LENGTHS = {"A": [5, 64, 90], "B": [1, 65, 100], "C": [41, 130, 200], "D": [7, 100]}
# Rounding to three bits behind the first one turns a difference of 2^-20 or so between two ways to a key or value into a step of
# 2^-3 of that number where it sits next to a border, about one number in 2^16: a step in one of a row's keys x head size products
# moves that row by far less than 1e-2 of its largest logit.  bfloat16 rows differ from the plain model by 2^-8, so more numbers
# (one in 2^5) go to the other side: as a whole like noise of one more rounding, 2^-4 / sqrt(2^5), on top of the usual tolerance.
F32_TOL, BF16_MORE = 1e-2, 2e-2


def engine(model_dirs, name, dtype, max_tokens=2048, cache_dtype="e4m3"):
    return sb.Engine(_load(str(model_dirs[name]), dtype), max_tokens=max_tokens, cache_dtype=cache_dtype)


@pytest.fixture
def rounded(monkeypatch):
    """The plain model with every page's keys and values of a head rounded to 8 bits."""
    real = pm.attention

    def by_page(x):
        out = x.clone()
        for at in range(0, x.shape[0], 64):
            for h in range(x.shape[1]):
                part = x[at:at + 64, h].double()
                scale = 2.0 ** plain.exponent_for(float(part.abs().max()))
                out[at:at + 64, h] = (plain.round_e4m3(part / scale) * scale).to(x.dtype)
        return out

    monkeypatch.setattr(pm, "attention", lambda q, k, v, *rest: real(q, by_page(k), by_page(v), *rest))


@pytest.mark.parametrize("name", list(TINY))
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_against_the_plain_model_with_rounded_keys_and_values(model_dirs, oracles, rounded, name, dtype):
    eng = engine(model_dirs, name, dtype)
    cfg, tensors = oracles[name]
    for p in prompts_for(name, LENGTHS[name]):
        err = pm.rel_err(whole(eng, p), pm.forward(cfg, tensors, p))
        assert err < (F32_TOL if dtype == "float32" else BF16_TOLS[name] + BF16_MORE), (len(p), err)
    eng.cache.check()


@pytest.mark.parametrize("name", list(TINY))
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_cuts_and_batches(model_dirs, name, dtype):
    """Tokens one by one, in unequal batches on pages that others left: as in one step.  (A page's scale depends on how far it is
    filled, which rounds numbers only below e4m3's normal range.)"""
    eng = engine(model_dirs, name, dtype)
    tol = F32_TOL if dtype == "float32" else BF16_TOLS[name] + BF16_MORE
    reqs = prompts_for(name, [70, 33, 100], seed=4)
    alone = [whole(eng, r) for r in reqs]
    for r, w in zip(reqs, alone):
        assert pm.rel_err(tail_one_by_one(eng, r, 32), w) < tol
    for got, w in zip(batch_unequal(eng, reqs, [64, 30, 1]), alone):
        assert pm.rel_err(got, w) < tol
    eng.cache.check()


def test_it_is_8_bits_that_are_read(model_dirs):
    p = prompts_for("B", [90])[0]
    a, b = (whole(engine(model_dirs, "B", "float32", cache_dtype=c), p) for c in (None, "e4m3"))
    assert 1e-4 < pm.rel_err(a, b) < 0.2


@pytest.mark.parametrize("name", ["A", "B", "C"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_the_captured_loop_gives_the_eager_tokens(model_dirs, name, dtype):
    """Its set-up run writes a token of no meaning at every current position: nothing of that may stay, not in the scales either."""
    prompts = prompts_for(name, [3, 61, 64], seed=2)
    outs = []
    for loop in (True, False):
        eng = engine(model_dirs, name, dtype)
        eng.use_decode_loop = loop
        model = llm.Model(eng.model)
        outs.append(llm.generate_batch(model, prompts, max_tokens=20, ignore_eos=True, engine=eng))
    assert outs[0] == outs[1]


def test_the_loops_set_up_run_leaves_pages_and_scales(model_dirs):
    eng = engine(model_dirs, "B", "bfloat16")
    slots = [eng.open(), eng.open()]
    eng.step([(slots[0], prompts_for("B", [70])[0], [69]), (slots[1], prompts_for("B", [5])[0], [4])])
    g = eng.cache.groups[0]
    before = g.storage.view(torch.uint8).clone(), g.scales.clone()
    from sonicboom_b200.sampling import Sampling
    loop = eng.decode_loop(slots, 10, [Sampling().checked()] * 2)
    assert torch.equal(before[0], g.storage.view(torch.uint8)) and torch.equal(before[1], g.scales)
    loop.close()


def test_sessions_and_prefix_reuse(model_dirs):
    model = llm.model_load(model_dirs["B"], dtype="bfloat16")
    p = prompts_for("B", [90], seed=6)[0]
    s = llm.session_new(model, 200, cache_dtype="e4m3")
    s.prefill(p)
    first = s.decode(llm.Sampling(max_tokens=12))
    assert s.prefill(p[:80] + p[:9]) == 80                                      # goes on in the middle of a page that held more
    again = s.decode(llm.Sampling(max_tokens=12))
    s.free()
    fresh = llm.session_new(model, 200, cache_dtype="e4m3")
    fresh.prefill(p[:80] + p[:9])
    assert fresh.decode(llm.Sampling(max_tokens=12)) == again and len(first) == 12
    fresh.free()
    assert llm.generate_batch(model, [p], max_tokens=12, ignore_eos=True, cache_dtype="e4m3")[0] == first


def test_layers_that_read_another_layers_cache(model_dirs):
    """A schedule whose second entry projects queries only."""
    from dataclasses import replace
    from sonicboom_b200.config.specs import ScheduleEntry
    base = _load(str(model_dirs["A"]), "float32")
    schedule = [ScheduleEntry(0), ScheduleEntry(1, cache_from=0)]
    try:
        spec = replace(base.spec, schedule=schedule)
    except TypeError:
        pytest.skip("the spec is no dataclass")
    model = sb.DecoderModel(spec, torch.float32, base.device)
    from sonicboom_b200.weights import RandomSource
    source = RandomSource(model.tensor_requests(), 3, 0.05, 0.1, 0.1, device=base.device)
    from sonicboom_b200.weights import fetch
    model.bind(lambda n: fetch(source, n, torch.float32, model.device))
    p = prompts_for("A", [70])[0]
    a, b = (whole(sb.Engine(model, 256, cache_dtype=c), p) for c in (None, "e4m3"))
    assert 1e-5 < pm.rel_err(a, b) < 0.2


def test_device_pages():
    from sonicboom_b200.cache import DevicePages
    pages = DevicePages(4, 6, 3, "cuda:0")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda:0")                  # noqa: E731
    slots, new = i32([2, 0]), i32([65, 3])
    t = pages.plan(slots, new, pages.tables(2, 70), 65)
    t.check()
    assert t.page_ids[:3].tolist() == [0, 1, 2] and t.page_off.tolist() == [0, 2, 3]
    pages.advance(slots, new, t)
    assert pages.lengths.tolist() == [3, 0, 65, 0] and int(pages.n_free) == 3
    pages.release(slots[:1])
    assert int(pages.n_free) == 5 and pages.free[:5].tolist() == [5, 4, 3, 0, 1] and pages.lengths.tolist() == [3, 0, 0, 0]


def test_the_command_line(model_dirs, tmp_path, capsys):
    from sonicboom_b200 import cli
    prompts = prompts_for("B", [5, 70], seed=9)
    tokens = tmp_path / "prompts.txt"
    tokens.write_text("\n".join(" ".join(map(str, p)) for p in prompts))
    assert cli.main(["generate", "-m", str(model_dirs["B"]), "--tokens", str(tokens), "-n", "6", "--ignore-eos", "--cache-dtype", "e4m3"]) == 0
    got = [[int(t) for t in line.split()] for line in capsys.readouterr().out.strip().splitlines()]
    model = llm.model_load(model_dirs["B"], dtype="bfloat16")
    assert got == llm.generate_batch(model, prompts, max_tokens=6, ignore_eos=True, cache_dtype="e4m3")


def test_a_graphs_scratch_outlives_a_larger_step():
    """Tables that a graph was captured with serve a step that needs more scratch memory: the graph's own stays."""
    from sonicboom_b200 import ops
    t = ops.PageTables(1, 4, 4, "cuda:0")
    a = t.scratch(100, "cuda:0")
    b = t.scratch(1000, "cuda:0")
    assert t.scratch(50, "cuda:0") is b and a.data_ptr() != b.data_ptr() and any(x is a for x in t._scratch)
