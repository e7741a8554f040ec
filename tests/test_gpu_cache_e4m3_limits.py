"""The 8-bit cache's kernels at the limits of what their calls say: lists that end too early, tokens that were taken back, scales far
apart, plans made on the device."""
import pytest
import torch

import plain_cache_e4m3 as plain
from sonicboom_b200 import ops
from test_gpu_cache_e4m3 import DEV, Plan

pytestmark = pytest.mark.gpu


def ones(n_pages, hkv, page, hd):
    return torch.ones(n_pages, 2, hkv, page, hd, device=DEV).to(torch.float8_e4m3fn), torch.ones(n_pages, 2, hkv, device=DEV)


@pytest.mark.parametrize("kernel,dtype,hd,page", [
    ("few", torch.bfloat16, 64, 64), ("few", torch.float32, 128, 64), ("values", torch.bfloat16, 64, 64), ("values", torch.bfloat16, 48, 64),
    ("values", torch.float32, 64, 64), ("values", torch.float32, 24, 64), ("values", torch.float32, 24, 16), ("plain", torch.bfloat16, 64, 64),
    ("plain", torch.float32, 22, 16)])
@pytest.mark.parametrize("n", [10, 1])
def test_a_sequence_whose_list_ends_among_its_new_rows_gets_zeros(kernel, dtype, hd, page, n):
    """All its rows, those before the list's end too, whatever kernel runs and whatever an earlier call left in scratch memory."""
    hq, hkv = 4, 2
    cache, scales = ones(4, hkv, page, hd)
    pos0 = page - 4
    for short in (False, True):                                                 # the first call leaves pages and numbers behind
        lists = [[0], [2, 3, 1]] if short and n > 1 else [[0, 1], [2, 3]]
        plan = Plan([n, 2], [pos0 if n > 1 else (2 * page if short else pos0), 5], lists)
        if short:
            plan._scratch = scratch
        plan.groups[0].page_size = page
        out = torch.full((n + 2, hq * hd), 5.0, dtype=dtype, device=DEV)
        ops.attention_e4m3(torch.ones(n + 2, hq, hd, dtype=dtype, device=DEV), out, plan, 0, cache, scales, hq, hkv, hd, 0, 0.1, kernel)
        scratch = plan._scratch
        # keys and values are ones: weights that add up to 1 give 1, to the roundings of at most 74 weights and of the result
        assert float((out[n:].float() - 1).abs().max()) <= 2.0 ** -7
        if short:
            assert bool((out[:n] == 0).all())
        else:
            assert float((out[:n].float() - 1).abs().max()) <= 2.0 ** -7


# ------------------------------------------------------------------------------------------------ tokens that are taken back
def test_a_prompt_that_goes_on_in_a_cut_page_is_as_a_fresh_one(model_dirs):
    """The page as a token far larger than the others would have left it, which is then cut away: its scale 2^20 times as large, the
    older numbers gone."""
    import plain_model as pm
    from conftest import prompts_for
    from sonicboom_b200 import llm
    from test_gpu_engine_e4m3 import F32_TOL
    model = llm.model_load(model_dirs["B"], dtype="float32")
    p = prompts_for("B", [90], seed=6)[0]
    sessions = [llm.session_new(model, 200, cache_dtype="e4m3") for _ in range(2)]
    sessions[0].prefill(p)
    g = sessions[0].engine.cache.groups[0]
    page = sessions[0].engine.cache.page_list(sessions[0].slot, 0)[1]
    g.scales[:, page] *= 2.0 ** 20
    g.storage.view(torch.uint8)[:, page] = 0
    logits, scales = [], []
    for s in sessions:
        s.prefill(p[:80] + p[:9])
        logits.append(s._logits.cpu())
        scales.append([s.engine.cache.groups[0].scales[:, i].cpu() for i in s.engine.cache.page_list(s.slot, 0)])
        assert s.engine.length(s.slot) == 89
        s.free()
    assert pm.rel_err(logits[0], logits[1]) < F32_TOL
    # a largest number within 2^-20 of a border would make a step of 2; none of these does
    assert all(torch.equal(a, b) for a, b in zip(*scales)) and len(scales[0]) == 2


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_a_retired_row_leaves_its_pages_alone(model_dirs, dtype):
    """The captured loop goes on for another row: the retired one's pages and scales stay, also where its last page is full or its
    budget is used up, and the sequence goes on from there as if nothing had been."""
    from conftest import prompts_for
    from sonicboom_b200.sampling import Sampling
    from test_gpu_engine_e4m3 import engine
    eng = engine(model_dirs, "B", dtype)
    slots, lengths, budgets = [eng.open() for _ in range(4)], [70, 61, 5, 9], [12, 3, 4, 30]
    eng.step([(s, p, [len(p) - 1]) for s, p in zip(slots, prompts_for("B", lengths, seed=3))])
    loop = eng.decode_loop(slots, budgets, [Sampling().checked()] * 4)
    tokens = [1, 2, 3, 4]
    for _ in range(3):                                                          # 73, 64 (a whole page, its budget used up) and 8 tokens
        tokens = loop.step_host(tokens)
    g = eng.cache.groups[0]
    before = g.storage.view(torch.uint8).clone(), g.scales.clone()
    for row in range(3):
        loop.retire(row)
    for _ in range(20):
        tokens = loop.step_host([7, 8, 9, tokens[3]])
    for i in range(3):
        pages = [p for p in eng.cache.page_list(slots[i], 0)]
        assert torch.equal(before[0][:, pages], g.storage.view(torch.uint8)[:, pages]) and torch.equal(before[1][:, pages], g.scales[:, pages])
    assert all(0 <= t for t in tokens[3:])
    loop.close()
    assert [eng.length(s) for s in slots] == [73, 64, 8, 32]


# ------------------------------------------------------------------------------------------------ plans made on the device
@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 64), (torch.float32, 64), (torch.float32, 22)])
def test_a_bfloat16_or_float32_cache_under_tables_made_on_the_device(dtype, hd):
    """`rope_store` and `attention` directly behind `page_tables`, eagerly and in a replayed graph, token by token across page ends:
    the same bits as with a plan from the host."""
    hq, hkv, n_pages = 4, 2, 8
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)                       # noqa: E731
    g = torch.Generator().manual_seed(hd)
    slots, new, lengths = i32([2, 0]), i32([1, 1]), i32([60, 9, 127])
    table, free, n_free = i32([[0, -1, -1], [-1] * 3, [1, 2, -1]]), i32([7, 6, 5, 4, 3, 0, 0, 0]), i32([5])
    caches = [torch.randn(n_pages, 2, hkv, 64, hd, generator=g).to(dtype).to(DEV) for _ in range(1)]
    caches.append(caches[0].clone())
    inv = torch.ones(hd // 2, device=DEV)
    t = ops.PageTables(2, 2, 6, DEV)
    x, q = torch.empty(2, (hq + 2 * hkv) * hd, device=DEV), torch.empty(2, hq, hd, dtype=dtype, device=DEV)
    outs = [torch.empty(2, hq * hd, dtype=dtype, device=DEV) for _ in range(2)]

    def one_step(plan, cache, out):
        group = plan.groups[0]
        ops.rope_store(x, hq, hkv, hd, 0, inv, plan.row_seq, plan.row_pos, group.page_off, group.page_ids, 64, cache, q)
        ops.attention(q, out, plan, 0, cache, hq, hkv, hd, 0, 0.125)

    def device_step():
        ops.page_tables(slots, new, lengths, table, free, n_free, t, 1, 192)
        one_step(t, caches[0], outs[0])
        ops.page_advance(slots, new, lengths, n_free, t)

    state = [caches[0], lengths, table, n_free]
    kept = [v.clone() for v in state]
    x.zero_()
    before = ops.LAUNCHES
    device_step()                                                               # builds what is built lazily; nothing of it stays
    assert ops.LAUNCHES - before == 5                                           # the one that keeps them apart among them
    torch.cuda.synchronize()
    for v, was in zip(state, kept):
        v.copy_(was)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        device_step()
    pages, pos = [[1, 2], [0]], [127, 60]
    for step in range(12):
        x.copy_(torch.randn(x.shape, generator=g))
        device_step() if step % 3 == 2 else graph.replay()
        for i in range(2):
            if pos[i] % 64 == 0:
                pages[i].append(3 + sum(len(p) for p in pages) - 3)             # the stack's top: 3, then 4, ...
        plan = Plan([1, 1], pos, pages)
        plan.max_len = 192
        one_step(plan, caches[1], outs[1])
        pos = [p + 1 for p in pos]
        assert torch.equal(outs[0], outs[1]) and torch.equal(caches[0], caches[1]), step
        assert lengths.tolist() == [pos[1], 9, pos[0]]


# ------------------------------------------------------------------------------------------------ how far numbers may lie apart
@pytest.mark.parametrize("kernel", ["few", "plain", "values"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("apart", [10, 29, 35, 50])
def test_pages_whose_scales_lie_far_apart(kernel, dtype, apart):
    """One page has 2^apart in its first channel, another one, that the same warp takes after it, 1 in its second; every key counts
    alike.  Weights times scales are halves in the "few" kernel: within 2^-40 of the largest, whatever the other page's is."""
    hq = hkv = 1
    hd, n_pages, length = 64, 36, 2200                                          # splits of eight pages from 2,049 keys on
    cache = torch.zeros(n_pages, 2, hkv, 64, hd, device=DEV)
    scales = torch.full((n_pages, 2, hkv), 2.0 ** -126, device=DEV)
    for page, channel, e in ((0, 0, apart - 8), (4, 1, -8)):
        cache[page, 1, 0, :, channel] = 256.0
        scales[page, 1] = 2.0 ** e
    plan = Plan([1], [length - 1], [list(range(-(-length // 64)))])
    out = torch.empty(1, hd, dtype=dtype, device=DEV)
    ops.attention_e4m3(torch.ones(1, 1, hd, dtype=dtype, device=DEV), out, plan, 0, cache.to(torch.float8_e4m3fn), scales, hq, hkv, hd, 0, 0.0, kernel)
    got, share = out.double().cpu()[0], 64 / length
    # sums in 32 bits of `length` terms and the result's rounding; a page's 64 weights are off by 2^-40 of the largest, which is 2^apart
    rounding = 2.0 ** -8 * (dtype == torch.bfloat16) + 2 * length * 2.0 ** -24
    weight = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -20               # relative, of a weight that is a normal number
    assert abs(float(got[0]) - share * 2.0 ** apart) <= (rounding + weight) * share * 2.0 ** apart
    lost = share * 2.0 ** (apart - 40) if kernel == "few" else 0.0
    assert abs(float(got[1]) - share) <= (rounding + weight) * share + lost
    assert bool((got[2:] == 0).all())


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dtype,kernel", [(torch.bfloat16, "values"), (torch.float32, "values"), (torch.float32, "plain"), (torch.bfloat16, "plain")])
@pytest.mark.parametrize("hd", [64, 48])
def test_a_nan_among_many_new_rows(dtype, kernel, kind, hd):
    """Every row that sees it becomes NaN, no row of another sequence; a row before it only where bfloat16 rows run over values and it
    is a value's."""
    hq, hkv, n, pos0, bad = 4, 2, 40, 70, 90
    cache, scales = ones(4, hkv, 64, hd)
    cache.view(torch.uint8)[1, kind, 0, bad - 64, 5] = 0x7f
    plan = Plan([n, n], [pos0, pos0], [[0, 1], [2, 3]])
    out = torch.empty(2 * n, hq * hd, dtype=dtype, device=DEV)
    ops.attention_e4m3(torch.ones(2 * n, hq, hd, dtype=dtype, device=DEV), out, plan, 0, cache, scales, hq, hkv, hd, 0, 0.1, kernel)
    got = out.view(2 * n, hq, hd).float().cpu()
    sees = torch.arange(pos0, pos0 + n) >= bad
    seen = got[:n, :2][sees]
    assert bool((seen if kind == 0 else seen[..., 5]).isnan().all())
    fine = torch.ones(2 * n, hq, hd, dtype=torch.bool)
    fine[:n, :2] = ~sees[:, None, None]
    if kind == 1:
        fine[..., [d for d in range(hd) if d != 5]] = True
        if dtype == torch.bfloat16 and kernel == "values":
            fine[:n, :2, 5] = False
    assert float((got[fine] - 1).abs().max()) <= 2.0 ** -7
