"""Calls at the edges of what the operators of the cache in eight bits allow: bounds that lie above the counts, as many
prompts as there can be, values of nothing beside small ones, scores and values far apart.  Tolerances count the roundings that test_quantized_cache_gpu.py names."""
import math

import numpy as np
import pytest
import torch

from llmx_b200 import ops
from test_quantized_cache_gpu import BF16, DEV, F32, Case, gpu, quantized, random_tree


# Heads of 64 and 128, queries of both types, up to 16, 32 and more (row, head) pairs (those of bfloat16 over heads of 128 by tcgen05), many rows.
FORMS = [(BF16, 4, 2, 128, 1), (BF16, 8, 1, 128, 3), (BF16, 8, 2, 128, 20), (BF16, 4, 2, 64, 3), (F32, 4, 2, 128, 2), (F32, 4, 2, 64, 30), (BF16, 8, 2, 128, 90),
         (BF16, 6, 3, 96, 3)]


class Done(Case):
    """A case whose outputs are there already."""
    def run(self, window=None):
        return self.done


def close(c, got, r, weight_step, least, window=None):
    """Request r's rows of `got` (float64) against 64 bits: a weight's rounding is `weight_step` of it, and `least` of the largest product
    of a row and head for each key that it sees."""
    n, h = c.requests[r]
    half_step = 2.0 ** -8 if c.dtype is BF16 else 2.0 ** -24
    kv, ok = c.keys(r), c.seen(r, window)
    for head in range(c.heads):
        k, v = (kv[:, plane, head // (c.heads // c.g)] for plane in (0, 1))
        x = c.q[c.starts[r]:c.starts[r] + n, head * c.dim:(head + 1) * c.dim].double()
        s = (x @ k.T * c.scale).masked_fill(~ok, -math.inf)
        w = torch.softmax(s, dim=-1)
        o, size = w @ v, w @ v.abs()
        score_error = (c.dim + 8) * 2.0 ** -24 * c.scale * torch.where(ok, x.abs() @ k.abs().T, 0.0).amax(-1, keepdim=True)
        largest = (w[:, :, None] * v.abs().amax(-1)[None, :, None]).amax(1) * ok.sum(-1, keepdim=True)
        limit = half_step * o.abs() + size * (2 * score_error + weight_step + (n + h + 16) * 2.0 ** -23) + least * largest
        mine = got[c.starts[r]:c.starts[r] + n, head * c.dim:(head + 1) * c.dim]
        bad = ~((mine - o).abs() <= limit)
        assert not bool(bad.any()), (r, head, bad.nonzero()[:4].tolist(), mine[bad][:4], o[bad][:4], limit[bad][:4])


# ---- a request of fewer rows than the call's bound ------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("n", [1, 10, 64, 65, 100])
@pytest.mark.parametrize("h", [0, 1500])
@pytest.mark.parametrize("window", [None, 70])
def test_one_request_of_fewer_rows_than_the_bound(n, h, window):
    """100 rows at most, of which the device's count names n.  Weights are bfloat16 where the bound is a prompt's."""
    c = Case([(n, h)], 8, 2, 128, 16, BF16, seed=21, spare_rows=100 - n)
    q, out = c.q.to(DEV), torch.full_like(c.q.to(DEV), 7.0)
    ops.attention_quantized(q, c.cache, out, *c.device(), c.heads, c.g, c.dim, window, c.scale, 100, 100 + h)
    assert bool((out[n:] == 7.0).all())
    close(c, out.double().cpu(), 0, 2.0 ** -8, 0.0, window)


@gpu
@pytest.mark.parametrize("window", [None, 70])
def test_one_request_recorded_at_the_bound_and_replayed_with_fewer_rows(window):
    c = Case([(100, 800)], 8, 2, 128, 16, BF16, seed=22, spare_rows=0)
    q, out = c.q.to(DEV), torch.zeros_like(c.q.to(DEV))
    start, count, history, tables = c.device()

    def call():
        ops.attention_quantized(q, c.cache, out, start, count, history, tables, c.heads, c.g, c.dim, window, c.scale, 100, 900)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for n, h in ((100, 800), (1, 800), (64, 33), (10, 0), (65, 700), (0, 50), (100, 800)):
        count.fill_(n)
        history.fill_(h)
        out.fill_(7.0)
        graph.replay()
        assert bool((out[n:] == 7.0).all())
        c.requests = [(n, h)]
        close(c, out.double().cpu(), 0, 2.0 ** -8, 0.0, window)


# ---- as many prompts as the rows make -----------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("requests", [[(17, 400)] * 20, [(300, 500)] + [(1, 700)] * 40, [(1, 90)] * 20 + [(17, 30), (0, 9), (19, 600)], [(16, 100)] * 20 + [(17, 0)] * 3])
@pytest.mark.parametrize("window", [None, 70])
def test_prompts_of_as_few_rows_as_are_expanded(requests, window):
    """64 pairs, of 4 heads, are the few-row form's; 17 rows are a prompt, and the room is for as many of them as there are rows."""
    Case(requests, 8, 2, 128, 16, BF16, seed=31, spare_rows=0).check(window)


@gpu
def test_prompts_that_name_the_same_rows():
    """More of them than their rows make: what does not fit is left out, and the rows are those of one that does."""
    c = Case([(70, 400)], 8, 2, 128, 16, BF16, seed=32, spare_rows=0)
    q, out = c.q.to(DEV), torch.full_like(c.q.to(DEV), 7.0)
    start, count, history, tables = (x.repeat_interleave(3, dim=0) for x in c.device())
    ops.attention_quantized(q, c.cache, out, start, count, history, tables, c.heads, c.g, c.dim, None, c.scale, 70, 470)
    close(c, out.double().cpu(), 0, 2.0 ** -8, 0.0)


# ---- values of nothing beside small ones --------------------------------------------------------------------------------------------------
def shift_values(c, by):
    c.cache.exponents[:, 1] = (c.cache.exponents[:, 1].int() + by).to(torch.uint8)
    c.values[:, 1] *= 2.0 ** by


def clear_values(c, where, negative=False):
    """Zeros (of either sign, as a row of them is written) as the values of slots `where` [pages, page], all heads."""
    at = where[:, None, :].expand(-1, c.g, -1)
    codes = c.cache.codes.view(torch.uint8)[:, 1]
    codes[at.to(DEV)] = 0x80 if negative else 0
    c.cache.exponents[:, 1][at.to(DEV)] = 127
    c.values[:, 1][at] = 0.0


@gpu
@pytest.mark.parametrize("dtype, heads, g, dim, n", FORMS)
@pytest.mark.parametrize("by", [-8, -20, -38])
@pytest.mark.parametrize("negative", [False, True])
def test_values_that_are_zeros_leave_the_others_their_bits(dtype, heads, g, dim, n, by, negative):
    c = Case([(n, 700), (1, 40)], heads, g, dim, 16, dtype, seed=23)
    shift_values(c, by)
    clear_values(c, torch.rand(c.pages, 16, generator=torch.Generator().manual_seed(1)) < 0.2, negative)
    c.check()


@gpu
@pytest.mark.parametrize("dtype, heads, g, dim, n", FORMS)
@pytest.mark.parametrize("by", [-8, -38])
def test_pages_that_are_not_there_leave_the_others_their_bits(dtype, heads, g, dim, n, by):
    c = Case([(n, 700), (1, 40)], heads, g, dim, 16, dtype, seed=24)
    shift_values(c, by)
    c.tables[0, 3], c.tables[0, 0], c.tables[0, 40] = -1, c.pages, -7
    c.check()


@gpu
@pytest.mark.parametrize("dtype, heads, g, dim, n", FORMS)
def test_tiles_of_zeros_before_values(dtype, heads, g, dim, n):
    """The first 300 keys' values are zeros, and all of the second request's: zeros, whatever the scores."""
    c = Case([(n, 700), (2, 40)], heads, g, dim, 16, dtype, seed=25)
    shift_values(c, -30)
    where = torch.zeros(c.pages, 16, dtype=torch.bool)
    for r, t in ((0, torch.arange(300)), (1, torch.arange(42))):
        where[c.tables[r].long()[t // 16], t % 16] = True
    clear_values(c, where)
    got = c.run()
    assert bool((got[n:] == 0).all())
    c.check()


@gpu
@pytest.mark.parametrize("dtype, heads, g, dim, n", FORMS[:6])
def test_trees_over_values_that_are_zeros(dtype, heads, g, dim, n):
    requests = [(n, 300), (5, 0), (2, 40)]
    c = Case(requests, heads, g, dim, 16, dtype, seed=26)
    c.tree = random_tree(requests, 26)
    shift_values(c, -30)
    clear_values(c, torch.rand(c.pages, 16, generator=torch.Generator().manual_seed(2)) < 0.3)
    c.check()


# ---- scores and values far apart ----------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype, heads, g, dim, n", FORMS[:6])
@pytest.mark.parametrize("at", [40, 200])
@pytest.mark.parametrize("apart", [60, 104])
def test_scores_that_rise_where_values_fall(dtype, heads, g, dim, n, at, apart):
    """Keys from `at` on have scores higher by `apart` (to base 2) and values smaller by as many powers: what they weigh together is
    much alike, and the sums of weights are not."""
    c = Case([(n, 500)], heads, g, dim, 16, dtype, seed=27, spread=0.0)
    c.scale = 1.0
    c.q.zero_()
    c.q.view(-1, heads, dim)[:, :, 0] = 1.0
    codes, b = c.cache.codes.view(torch.uint8), c.cache.exponents
    # A key's first value is its score: eighths around nought, from `at` on eights up to what `apart` is to base e.
    steps = round(apart * math.log(2) / 8.0)
    t = torch.arange(n + 500)
    page, place = c.tables[0].long()[t // 16], t % 16
    key = torch.zeros(len(t), dim)
    key[:, 0] = torch.randn(len(t), generator=torch.Generator().manual_seed(3)).mul(4).round().clamp(-7, 7) / 8
    key[at:, 0] = 8.0 * steps
    values, e = quantized(key.double().numpy())
    raw = torch.from_numpy(values).float().to(torch.float8_e4m3fn).view(torch.uint8)
    low = round(apart / 2)
    for head in range(g):
        codes[page.to(DEV), 0, head, place.to(DEV)] = raw.to(DEV)
        b[page.to(DEV), 0, head, place.to(DEV)] = torch.from_numpy(e).to(torch.uint8).to(DEV)
        c.values[page, 0, head, place] = torch.from_numpy(values * np.exp2(e[:, None] - 127.0))
        for part, by in ((t < at, low), (t >= at, -low)):
            b[page[part].to(DEV), 1, head, place[part].to(DEV)] = (b[page[part].to(DEV), 1, head, place[part].to(DEV)].int() + by).to(torch.uint8)
            c.values[page[part], 1, head, place[part]] *= 2.0 ** by
    c.check()


# ---- sizes beside the usual ones ----------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("heads, g, dim", [(8, 2, 128), (4, 2, 64), (5, 1, 64)])
@pytest.mark.parametrize("requests", [[(300, 0)], [(300, 200), (1, 90), (40, 33)]])
@pytest.mark.parametrize("window", [None, 70])
def test_prompts_with_queries_of_32_bits(heads, g, dim, requests, window):
    Case(requests, heads, g, dim, 16, F32, seed=41).check(window)


@gpu
@pytest.mark.parametrize("page", [48, 112, 512, 528])
@pytest.mark.parametrize("dtype, heads, g, dim, n", FORMS[:7])
def test_pages_of_other_sizes(page, dtype, heads, g, dim, n):
    Case([(n, 1100), (1, 3), (2, page)], heads, g, dim, page, dtype, seed=page).check()


@gpu
@pytest.mark.parametrize("page", [48, 512])
@pytest.mark.parametrize("heads, g, dim, n", [(8, 2, 128, 1), (8, 2, 128, 6), (8, 2, 128, 20), (4, 2, 64, 9)])
def test_trees_over_bfloat16_pages_of_other_sizes(page, heads, g, dim, n):
    requests = [(n, 1100), (3, 0), (2, page)]
    c = Case(requests, heads, g, dim, page, BF16, "bfloat16", seed=page)
    c.tree = random_tree(requests, page, words=3)
    c.check()


@gpu
@pytest.mark.parametrize("dtype, heads, g, dim, n", FORMS)
@pytest.mark.parametrize("tree", [False, True])
def test_bounds_far_above_what_there_is(dtype, heads, g, dim, n, tree):
    """As a program says them that records one call for all that may come."""
    class Loose(Case):
        def bounds(self):
            return 150, 20000
    c = Loose([(n, 300), (0, 9), (1, 40), (2, 0)], heads, g, dim, 16, dtype, seed=42, spare_rows=200)
    if tree:
        c.tree = np.concatenate([random_tree(c.requests, 42, words=5), np.zeros((198, 5), dtype=np.int32)])
    c.check()


@gpu
@pytest.mark.parametrize("n", [1, 3])
def test_many_requests(n):
    """More than a warp's lanes, of all lengths, none among them."""
    gen = np.random.default_rng(43)
    requests = [(int(gen.integers(0, n + 1)), int(gen.integers(0, 90))) for _ in range(300)]
    Case(requests, 4, 2, 128, 16, BF16, seed=43).check()
    Case(requests, 4, 2, 64, 16, F32, seed=44).check()


@gpu
def test_calls_on_two_streams_at_once():
    cases = [Case([(1, 3000), (2, 700)], 8, 2, 128, 16, BF16, seed=45), Case([(20, 900)], 8, 2, 128, 16, BF16, seed=46), Case([(200, 700)], 8, 2, 128, 16, BF16, seed=47),
             Case([(2, 900)], 4, 2, 64, 16, F32, seed=48)]
    wants = [c.run() for c in cases]
    ready = [(c, c.q.to(DEV), c.device()) for c in cases]
    outs = [torch.full_like(q, 7.0) for _ in range(2) for _, q, _ in ready]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for stream in streams:
        stream.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for i in range(len(outs)):
            c, q, rows = ready[i % len(ready)]
            with torch.cuda.stream(streams[(i + i // len(ready)) % 2]):
                ops.attention_quantized(q, c.cache, outs[i], *rows, c.heads, c.g, c.dim, None, c.scale, *c.bounds())
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        c = cases[i % len(cases)]
        assert torch.equal(out[:c.rows].double().cpu(), wants[i % len(cases)])


# ---- an invariant engine ------------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("name", ["A", "D", "E"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_an_invariant_engine_over_eight_bits_gives_a_row_the_same_bits_in_any_batch(model_dirs, name, dtype):
    import helpers
    from configs import CONFIGS
    from llmx_b200.engine import Engine, EngineOptions
    d16, d32, page = model_dirs[name]
    requests = {f"i{i}": helpers.random_ids(CONFIGS[name][0]["vocab_size"], n, seed=80 + i) for i, n in enumerate([70, 9, 40, 33, 81])}
    base = None
    for make in (helpers.trace_whole, helpers.trace_tail_decoded, helpers.trace_portions, helpers.trace_mixed):
        steps = make(requests)
        engine = Engine.from_dir(d32 if dtype == "float32" else d16,
                                 EngineOptions(dtype=dtype, kv_dtype="float8_e4m3", kv_tokens=helpers.tokens_needed(steps), page_size=page, max_requests=4,
                                               invariant=True))
        got = helpers.run_trace(engine, steps)
        del engine
        base = base or got
        assert got.keys() == base.keys()
        moved = [k for k in base if not np.array_equal(base[k], got[k])]
        assert not moved, (make.__name__, len(moved), moved[:5])


# ---- places and rows anywhere -------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype, heads, g, dim, n", FORMS)
def test_a_cache_beyond_32_bits_of_bytes(dtype, heads, g, dim, n):
    """The same pages at the far end of a cache of more than 2^32 bytes: the same bits; written there, and read back."""
    c = Case([(n, 300), (1, 40)], heads, g, dim, 16, dtype, seed=51)
    want = c.run()
    pages = 2 ** 32 // (2 * g * 16 * dim) + c.pages + 5
    far = pages - c.pages
    large = ops.QuantizedPages.zeros(pages, g, 16, dim, DEV)
    large.codes[far:], large.exponents[far:] = c.cache.codes, c.cache.exponents
    small, c.cache = c.cache, large
    tables = c.tables
    c.tables = torch.where(tables >= 0, tables + far, tables)
    assert torch.equal(c.run(), want)
    ids = torch.tensor([pages - 1, far], dtype=torch.int32, device=DEV)
    for t in (F32, BF16):
        out = [torch.empty(2, 2, g, 16, dim, dtype=t, device=DEV) for _ in range(2)]
        ops.dequantize_pages(large, ids, out[0])
        ops.dequantize_pages(small, ids - far, out[1])
        assert torch.equal(*out)
    k, v = (torch.randn(40, g, dim, device=DEV) for _ in range(2))
    slots = torch.randperm(c.pages * 16, device=DEV)[:40].int()
    ops.quantize_kv(k, v, slots, small)
    ops.quantize_kv(k, v, slots + far * 16, large)
    assert torch.equal(large.codes[far:].view(torch.uint8), small.codes.view(torch.uint8)) and torch.equal(large.exponents[far:], small.exponents)


@gpu
@pytest.mark.parametrize("dtype, heads, g, dim, n", FORMS)
def test_storage_that_starts_anywhere(dtype, heads, g, dim, n):
    """Calls of one size whose queries, outputs, codes and exponents begin off their 16 bytes, in turn."""
    def moved(x, by):
        raw = torch.empty(x.numel() * x.element_size() + 64, dtype=torch.uint8, device=DEV)
        y = raw[by:by + x.numel() * x.element_size()].view(x.dtype).view(x.shape)
        y.copy_(x)
        return y

    c = Done([(n, 300), (1, 40)], heads, g, dim, 16, dtype, seed=52, spare_rows=0)
    codes, exponents = c.cache.codes, c.cache.exponents
    for what in ("q", "out", "codes", "exponents", ""):
        q, out = c.q.to(DEV), torch.zeros_like(c.q.to(DEV))
        if what == "q":
            q = moved(q, q.element_size())
        if what == "out":
            out = moved(out, out.element_size())
        cache = ops.QuantizedPages(moved(codes.view(torch.uint8), 1).view(torch.float8_e4m3fn) if what == "codes" else codes,
                                   moved(exponents, 1) if what == "exponents" else exponents)
        ops.attention_quantized(q, cache, out, *c.device(), c.heads, c.g, c.dim, None, c.scale, *c.bounds())
        c.done = out.double().cpu()
        c.check()


@gpu
@pytest.mark.parametrize("dtype, heads, g, dim, n", FORMS)
def test_rows_in_any_order_with_others_between(dtype, heads, g, dim, n):
    c = Done([(n, 300), (2, 40), (0, 7), (1, 20)], heads, g, dim, 16, dtype, seed=53, spare_rows=0)
    starts, at = [0] * 4, 3
    for r in (3, 1, 0, 2):
        starts[r] = at
        at += c.requests[r][0] + 2
    q, out = torch.randn(at, heads * dim, device=DEV).to(dtype), torch.full((at, heads * dim), 7.0, dtype=dtype, device=DEV)
    mine = torch.zeros(at, dtype=torch.bool)
    for r, (rows, _) in enumerate(c.requests):
        q[starts[r]:starts[r] + rows] = c.q[c.starts[r]:c.starts[r] + rows].to(DEV)
        mine[starts[r]:starts[r] + rows] = True
    _, count, history, tables = c.device()
    ops.attention_quantized(q, c.cache, out, torch.tensor(starts, dtype=torch.int32, device=DEV), count, history, tables, heads, g, dim, None, c.scale, *c.bounds())
    assert bool((out[~mine.to(DEV)] == 7.0).all())
    # (Not the bits of another order: rows of a tile are given new references together, whosever they are.)
    c.done = torch.cat([out[starts[r]:starts[r] + rows] for r, (rows, _) in enumerate(c.requests)]).double().cpu()
    c.check()


@gpu
@pytest.mark.parametrize("store", ["e4m3", "bfloat16"])
@pytest.mark.parametrize("dtype, heads, g, dim, n", [f for f in FORMS if f[-1] > 1])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_row_of_queries_that_are_no_numbers_is_its_own(store, dtype, heads, g, dim, n, bad):
    requests = [(n, 300), (2, 40)]
    c = Case(requests, heads, g, dim, 16, dtype, store, seed=54, spare_rows=0)
    if store == "bfloat16":
        c.tree = random_tree(requests, 54)[:n + 2]
        c.tree[1] = 1                                    # (sees something)
    want, q = c.run(), c.q.clone()
    c.q[1, :2 * dim] = bad
    got, c.q = c.run(), q
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[1, :2 * dim] = True
    assert bool(got[hit].isnan().all())
    # (Not the same bits: a warp's rows are given new references together, when one of them needs it.)
    c.done = torch.where(hit, want, got)
    c.__class__ = Done
    c.check()
