"""The cache in eight bits, read and written, and attention over it and for trees of drafted tokens, against plain forms in 64 bits.

Tolerances.  Writing and reading back round once, to values that can be named: they are compared for equality.  Attention's
output o = sum w v is off by
    half a step of its type (bfloat16 2^-8, float32 2^-24 of |o|),
    a score's error, twice (a weight's numerator and the sum that divides it), times A = sum w |v|: D products and their sum in 32
    bits, (D + 8) 2^-24 of scale * sum |q k|,
    a weight's rounding to half precision, 2^-11 of it, where queries are bfloat16, 2^-21 (two halves) where they are float32; to
    bfloat16, whose eight bits leave half a step of 2^-8, over a bfloat16 cache and where a request's many rows run the prompt
    kernel; and, of a weight that is small beside the row's largest, half of 2^-24 of the largest, for each key (heads of 128 with
    bfloat16 queries over eight bits: weights are three codes that add up, the third in steps of 2^-9 / 1024, half of which is
    2^-20 of the largest),
    the sums over the keys in 32 bits, (keys + 16) 2^-23."""
import math

import numpy as np
import pytest
import torch

from llmx_b200 import ops

gpu = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


# ---- writing and reading back -----------------------------------------------------------------------------------------------------------
def decoded(codes, exponents):
    """float64 values (numpy) of codes and exponents, from what the eight bits mean."""
    c = codes.cpu().view(torch.uint8).numpy().astype(np.int64)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * np.exp2(e - 10.0)) * np.where(c >= 128, -1.0, 1.0)
    b = exponents.cpu().numpy().astype(np.float64)[..., None]
    return np.where(b == 255, np.nan, v * np.exp2(b - 127))


def quantized(x):
    """float64 (values of codes, exponent bytes) of float64 rows [..., D], from the definition."""
    with np.errstate(invalid="ignore"):
        peak = np.abs(x).max(-1)
        bad = ~np.isfinite(x).all(-1)
        m, e = np.frexp(np.where(bad | (peak == 0), 1.0, peak))
        n = np.where(m <= 0.875, e - 9, e - 8).clip(-60, 60)
        n = np.where(peak == 0, 0, n)
        y = np.where(bad[..., None], 0.0, x) * np.exp2(-n.astype(np.float64))[..., None]
        y = y.clip(-448, 448)
        step = np.exp2(np.floor(np.log2(np.abs(y).clip(2.0 ** -6, None))) - 3)
        return np.rint(y / step) * step, np.where(bad, 255, n + 127)


def special_rows(dim, gen):
    """Rows at every border that the definition has."""
    rows = [np.zeros(dim), np.full(dim, 448.0), np.full(dim, 448.0 * (1 + 2.0 ** -7)), np.full(dim, 464.0 * 2.0 ** -20), np.full(dim, 2.0 ** -149),
            np.full(dim, 2.0 ** -60), np.full(dim, 3.0e38), np.full(dim, 1e-16), np.full(dim, 448.0 * 2.0 ** 60), np.full(dim, 2.0 ** -126)]
    for bad in (np.inf, -np.inf, np.nan):
        row = gen.standard_normal(dim)
        row[dim // 2] = bad
        rows.append(row)
    ties = (np.arange(dim) % 16 + 8.5) * 2.0 ** (np.arange(dim) % 5 - 2.0)       # halfway between codes, some of them
    ties[0] = 448.0
    rows.append(ties)
    small = np.exp2(-np.linspace(0, 30, dim)) * 300                              # down through the codes without a leading one
    rows.append(small * np.where(np.arange(dim) % 2, -1, 1))
    one = np.zeros(dim)
    one[-1] = -1e-3
    rows.append(one)
    return np.stack(rows)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim, page", [(128, 16), (64, 32), (100, 16), (256, 5), (1, 3), (48, 16), (33, 1)])
@pytest.mark.parametrize("strided", [False, True])
def test_write_and_read_back(dtype, dim, page, strided):
    gen = np.random.default_rng(dim * page + strided)
    g, rows = 3, 45
    k = gen.standard_normal((rows, g, dim)) * np.exp(2 * gen.standard_normal((rows, g, 1)))
    v = gen.standard_normal((rows, g, dim)) * np.exp(gen.standard_normal((rows, g, dim)))
    special = special_rows(dim, gen)
    k[:len(special), 0], v[-len(special):, g - 1] = special, special
    k, v = (torch.from_numpy(x).to(torch.float32).to(dtype).to(DEV) for x in (k, v))
    if strided:                       # columns of a wider matrix, that does not start on any boundary
        wide = torch.randn(rows, 2 * g * dim + 7, device=DEV).to(dtype)
        wide[:, 3:3 + g * dim], wide[:, 5 + g * dim:5 + 2 * g * dim] = k.reshape(rows, -1), v.reshape(rows, -1)
        k, v = wide[:, 3:3 + g * dim].view(rows, g, dim), wide[:, 5 + g * dim:5 + 2 * g * dim].view(rows, g, dim)
    n_pages = -(-rows // page) + 2
    cache = ops.QuantizedPages.zeros(n_pages, g, page, dim, DEV)
    cache.codes.view(torch.uint8).random_(0, 127)
    cache.exponents.random_(100, 140)
    codes, exponents = cache.codes.view(torch.uint8).cpu().numpy().copy(), cache.exponents.cpu().numpy().copy()
    before = decoded(cache.codes, cache.exponents)
    slots = torch.from_numpy(gen.permutation(n_pages * page)[:rows].astype(np.int32))
    slots[7], slots[20], slots[21], slots[22] = -1, n_pages * page, 2 ** 31 - 1, -2 ** 31
    ops.quantize_kv(k, v, slots.to(DEV), cache)
    want, want_exponents = before.copy(), exponents.copy()
    for plane, x in enumerate((k, v)):
        values, b = quantized(x.float().cpu().numpy().astype(np.float64))
        for r, slot in enumerate(slots.tolist()):
            if 0 <= slot < n_pages * page:
                want_exponents[slot // page, plane, :, slot % page] = b[r]
                want[slot // page, plane, :, slot % page] = np.where(b[r][:, None] == 255, np.nan, values[r] * np.exp2(b[r][:, None] - 127.0))
    assert np.array_equal(cache.exponents.cpu().numpy(), want_exponents)
    assert np.array_equal(decoded(cache.codes, cache.exponents), want, equal_nan=True)
    got = cache.codes.view(torch.uint8).cpu().numpy()
    assert not got[want_exponents == 255].any()                                  # no code is a NaN
    untouched = np.ones(got.shape[:4], dtype=bool)
    for slot in slots.tolist():
        if 0 <= slot < n_pages * page:
            untouched[slot // page, :, :, slot % page] = False
    assert np.array_equal(got[untouched], codes[untouched])

    # And back: pages in any order, one twice, ones that are not there, part of some.
    ids = [1, 0, n_pages - 1, 1, -1, n_pages, 0]
    used = [page, 0, page - 1, 1, page, page, page + 9]
    for out_type in (F32, BF16):
        for part in (None, used):
            out = torch.full((len(ids), 2, g, page, dim), 7.0, dtype=out_type, device=DEV)
            ops.dequantize_pages(cache, torch.tensor(ids, dtype=torch.int32, device=DEV), out,
                                 None if part is None else torch.tensor(part, dtype=torch.int32, device=DEV))
            wanted = np.zeros(out.shape)
            for i, p in enumerate(ids):
                if 0 <= p < n_pages:
                    n = page if part is None else min(page, part[i])
                    wanted[i, :, :, :n] = want[p, :, :, :n]
            assert np.array_equal(out.float().cpu().numpy().astype(np.float64), wanted, equal_nan=True)


@gpu
def test_write_and_read_nothing():
    cache = ops.QuantizedPages.zeros(2, 2, 16, 64, DEV)
    ops.quantize_kv(torch.empty(0, 2, 64, device=DEV), torch.empty(0, 2, 64, device=DEV), torch.empty(0, dtype=torch.int32, device=DEV), cache)
    out = torch.empty(0, 2, 2, 16, 64, device=DEV)
    assert ops.dequantize_pages(cache, torch.empty(0, dtype=torch.int32, device=DEV), out) is out


# ---- attention ------------------------------------------------------------------------------------------------------------------------------
class Case:
    """Requests (rows, history) over a shuffled cache whose unused slots hold what must not be read."""

    def __init__(self, requests, heads, g, dim, page, dtype, store="e4m3", seed=0, spare_rows=2, spread=1.0):
        gen = torch.Generator().manual_seed(seed)
        self.requests, self.heads, self.g, self.dim, self.page, self.dtype, self.store = requests, heads, g, dim, page, dtype, store
        need = [max(1, -(-(n + h) // page)) for n, h in requests]
        self.pages = sum(need) + 2
        order = torch.randperm(self.pages, generator=gen).int()
        width = max(need) + 1
        self.tables = torch.full((len(requests), width), -1, dtype=torch.int32)
        at = 0
        for r, n in enumerate(need):
            self.tables[r, :n] = order[at:at + n]
            at += n
        shape = (self.pages, 2, g, page)
        values = torch.randn(*shape, dim, generator=gen) * torch.exp(spread * torch.randn(*shape, 1, generator=gen))
        if store == "e4m3":
            codes, b = quantized(values.double().numpy())
            self.cache = ops.QuantizedPages(torch.from_numpy(codes).float().to(torch.float8_e4m3fn).to(DEV), torch.from_numpy(b).to(torch.uint8).to(DEV))
            self.values = torch.from_numpy(codes * np.exp2(b[..., None] - 127.0))
        else:
            self.cache = values.to(getattr(torch, store)).to(DEV)
            self.values = self.cache.double().cpu()
        self.starts, at = [], 0
        for n, _ in requests:
            self.starts.append(at)
            at += n
        self.rows = at
        self.q = torch.randn(at + spare_rows, heads * dim, generator=gen).to(dtype)
        self.scale = 1 / math.sqrt(dim)
        self.tree = None

    def device(self):
        def ints(x):
            return torch.tensor(x, dtype=torch.int32, device=DEV)
        return (ints(self.starts), ints([n for n, _ in self.requests]), ints([h for _, h in self.requests]), self.tables.to(DEV))

    def bounds(self):
        return max(n for n, _ in self.requests), max(n + h for n, h in self.requests)

    def run(self, window=None, out=None):
        q = self.q.to(DEV)
        out = torch.full_like(q, 7.0) if out is None else out
        if self.tree is None:
            ops.attention_quantized(q, self.cache, out, *self.device(), self.heads, self.g, self.dim, window, self.scale, *self.bounds())
        else:
            ops.attention_tree(q, self.cache, out, *self.device(), torch.from_numpy(self.tree).to(DEV), self.heads, self.g, self.dim, self.scale,
                               *self.bounds())
        assert bool((out[self.rows:] == 7.0).all()), "rows of no request were written"
        return out[:self.rows].double().cpu()

    def keys(self, r):
        n, h = self.requests[r]
        t = torch.arange(n + h)
        page = self.tables[r].long()[t // self.page]
        v = self.values[page.clamp(0, self.pages - 1), :, :, t % self.page]
        return torch.where(((page >= 0) & (page < self.pages))[:, None, None, None], v, 0.0)       # [keys, 2, g, dim]

    def seen(self, r, window=None):
        n, h = self.requests[r]
        t, i = torch.arange(n + h)[None], torch.arange(n)[:, None]
        if self.tree is None:
            ok = t <= h + i
            return ok & (t > h + i - window) if window else ok
        words = torch.from_numpy(self.tree.view(np.uint32)[self.starts[r]:self.starts[r] + n].astype(np.int64))
        j = (t - h).clamp(min=0).expand(n, -1)
        inside = j // 32 < words.shape[1]
        bit = (words.gather(1, (j // 32).clamp(max=words.shape[1] - 1)) >> (j % 32)) & 1
        return (t < h) | ((bit == 1) & inside)

    def check(self, window=None, **kw):
        got = self.run(window, **kw)
        half_step = 2.0 ** -8 if self.dtype is BF16 else 2.0 ** -24
        for r, (n, h) in enumerate(self.requests):
            if n == 0:
                continue
            most = 64 * min(4, max(1, 32 // (len(self.requests) * self.g)))       # pairs of a request whose weights are not rounded to bfloat16
            prompt = self.tree is None and self.dim == 128 and n * self.heads // self.g > most
            weight_step = 2.0 ** -21 if self.dtype is F32 else 2.0 ** -8 if self.store == "bfloat16" or prompt else 2.0 ** -11
            kv, ok = self.keys(r), self.seen(r, window)
            for head in range(self.heads):
                k, v = kv[:, 0, head // (self.heads // self.g)], kv[:, 1, head // (self.heads // self.g)]
                x = self.q[self.starts[r]:self.starts[r] + n, head * self.dim:(head + 1) * self.dim].double()
                s = (x @ k.T * self.scale).masked_fill(~ok, -math.inf)
                w = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300))
                w = torch.where(ok, w, 0.0)
                total = w.sum(-1, keepdim=True)
                w = w / torch.where(total == 0, 1.0, total)
                v = torch.where(ok.any(0)[:, None], v, 0.0)
                o = w @ v
                score_error = (self.dim + 8) * 2.0 ** -24 * self.scale * torch.where(ok, x.abs() @ k.abs().T, 0.0).amax(-1, keepdim=True)
                size = w @ v.abs()
                # The weights that multiply the values carry the values' powers of two: it is the largest product that counts.
                codes = self.store == "e4m3" and self.dim == 128 and self.dtype is BF16 and not prompt
                least = (2.0 ** -20 if codes else 2.0 ** -24 * min(1.0, weight_step / 2.0 ** -11)) * (w[:, :, None] * v.abs().amax(-1)[None, :, None]).amax(1) * ok.sum(-1, keepdim=True)
                limit = half_step * o.abs() + size * (2 * score_error + weight_step + (n + h + 16) * 2.0 ** -23) + least + 1e-30
                mine = got[self.starts[r]:self.starts[r] + n, head * self.dim:(head + 1) * self.dim]
                bad = ~((mine - o).abs() <= limit)
                assert not bool(bad.any()), (r, head, bad.nonzero()[:4].tolist(), mine[bad][:4], o[bad][:4], limit[bad][:4])


MIXED = [(1, 0), (1, 511), (3, 0), (2, 64), (1, 31), (17, 100), (0, 40), (1, 1000)]
SHAPES = [(8, 2, 128, 16), (4, 4, 64, 16), (10, 2, 128, 32), (16, 1, 64, 16), (40, 2, 128, 16), (6, 3, 96, 16), (4, 2, 128, 5), (2, 1, 32, 16), (2, 2, 256, 16)]


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads, g, dim, page", SHAPES)
@pytest.mark.parametrize("window", [None, 1, 70])
def test_attention_over_eight_bits(dtype, heads, g, dim, page, window):
    Case(MIXED, heads, g, dim, page, dtype, seed=heads).check(window)


@gpu
@pytest.mark.parametrize("heads, g, dim", [(8, 2, 128), (4, 2, 64), (8, 8, 128), (20, 4, 128)])
@pytest.mark.parametrize("requests", [[(1, 5000)], [(1, 0)], [(1, 2047), (1, 3)], [(1, n) for n in range(29, 35)], [(4, 4096)], [(7, 777), (1, 2900)],
                                      [(33, 1000)], [(64, 200), (1, 100)]])
def test_attention_over_eight_bits_of_few_rows(heads, g, dim, requests):
    Case(requests, heads, g, dim, 16, BF16, seed=1, spread=2.0).check()


@gpu
@pytest.mark.parametrize("heads, g, dim", [(8, 2, 128), (4, 4, 128), (5, 1, 128), (4, 2, 64)])
@pytest.mark.parametrize("requests", [[(300, 0)], [(257, 700)], [(200, 33), (1, 900), (130, 0), (2, 64)], [(129, 1500), (0, 7), (500, 16)]])
@pytest.mark.parametrize("window", [None, 100])
def test_attention_over_eight_bits_of_prompts(heads, g, dim, requests, window):
    Case(requests, heads, g, dim, 16, BF16, seed=2).check(window)


def random_tree(requests, seed, words=None, share=0.5):
    """Any bits at all: rows that see tokens behind them, rows that see none (not even themselves)."""
    rng = np.random.default_rng(seed)
    words = max(1, -(-max(n for n, _ in requests) // 32)) if words is None else words
    rows = sum(n for n, _ in requests) + 2
    bits = np.zeros((rows, words), dtype=np.uint32)
    for b in range(32):
        bits |= (rng.random((rows, words)) < share).astype(np.uint32) << np.uint32(b)
    bits[::5] = 0
    return bits.view(np.int32)


@gpu
@pytest.mark.parametrize("store", ["e4m3", "bfloat16", "float32"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads, g, dim, page", SHAPES)
def test_tree_of_any_bits(store, dtype, heads, g, dim, page):
    requests = [(5, 0), (1, 0), (17, 100), (0, 3), (40, 31), (2, 600)]
    c = Case(requests, heads, g, dim, page, dtype, store, seed=dim)
    c.tree = random_tree(requests, dim)
    c.check()


@gpu
@pytest.mark.parametrize("store", ["e4m3", "bfloat16"])
@pytest.mark.parametrize("heads, g, dim", [(32, 8, 128), (4, 2, 64), (3, 3, 128)])
@pytest.mark.parametrize("requests", [[(2, 0)], [(64, 3000)], [(16, 400), (9, 1000), (31, 15)], [(150, 77)], [(1, 2000), (1, 10)]])
def test_trees_that_grow(store, heads, g, dim, requests):
    rng = np.random.default_rng(3)
    c = Case(requests, heads, g, dim, 16, BF16, store, seed=3, spare_rows=0)
    c.tree = ops.tree_bits([[int(rng.integers(-1, i)) if i else -1 for i in range(n)] for n, _ in requests])
    c.check()


@gpu
def test_a_tree_that_is_a_chain_is_what_decoding_sees():
    requests = [(9, 300), (4, 0), (1, 77)]
    c = Case(requests, 8, 2, 128, 16, BF16, seed=4)
    plain = c.run()
    c.tree = np.concatenate([ops.tree_bits([list(range(-1, n - 1)) for n, _ in requests]), np.zeros((2, 1), dtype=np.int32)])
    assert float((c.run() - plain).abs().max()) <= 2.0 ** -7 * float(plain.abs().max())


@gpu
def test_fewer_words_than_rows_hide_the_rows_behind():
    requests = [(40, 20)]
    c = Case(requests, 4, 2, 128, 16, BF16, seed=5)
    c.tree = random_tree(requests, 5, words=1)
    c.check()


@gpu
@pytest.mark.parametrize("heads, g, dim, page", [(8, 2, 128, 16), (4, 2, 64, 32), (4, 2, 96, 16)])
@pytest.mark.parametrize("rows", [1, 20, 200])
def test_slots_behind_the_last_key_and_below_the_window_are_not_read(heads, g, dim, page, rows):
    """Codes that are NaN and exponents that are none, in every slot that no row sees."""
    c = Case([(rows, 333), (1, 5)], heads, g, dim, page, BF16, seed=6)
    window = 50
    live = torch.zeros(c.pages, page, dtype=torch.bool)
    for r, (n, h) in enumerate(c.requests):
        t = torch.arange(max(0, h - window + 1), n + h)
        live[c.tables[r].long()[t // page], t % page] = True
    dead = ~live[:, None, None, :].expand(-1, 2, g, -1)
    c.cache.codes.view(torch.uint8)[dead.to(DEV)] = 0x7F
    c.cache.exponents[dead.to(DEV)] = 255
    c.check(window)


@gpu
@pytest.mark.parametrize("store", ["e4m3", "bfloat16"])
@pytest.mark.parametrize("plane", [0, 1])
def test_rows_that_do_not_see_a_drafted_token_do_not_meet_its_infinities(store, plane):
    requests = [(6, 40), (3, 10)]
    c = Case(requests, 4, 2, 128, 16, BF16, store, seed=7, spare_rows=0)
    c.tree = ops.tree_bits([[-1, 0, 0, 1, 2, 2], [-1, 0, 1]])
    want = c.run()
    page, place = int(c.tables[0][42 // 16]), 42 % 16                        # request 0, its third token
    if store == "e4m3":
        k = torch.randn(1, 2, 128, device=DEV)
        k[0, :, 5] = math.inf
        other = torch.zeros_like(k)
        slot = torch.tensor([page * 16 + place], dtype=torch.int32, device=DEV)
        ops.quantize_kv(*((k, other) if plane == 0 else (other, k)), slot, c.cache)
    else:
        c.cache[page, plane, :, place] = math.nan
    got = c.run()
    sees = [2, 4, 5]
    others = [i for i in range(9) if i not in sees]
    assert torch.equal(got[others], want[others])
    assert bool(got[sees].isnan().all())


@gpu
@pytest.mark.parametrize("store, dtype, heads, g, dim", [("bfloat16", BF16, 4, 2, 128), ("bfloat16", BF16, 4, 2, 64), ("bfloat16", BF16, 4, 2, 96),
                                                         ("bfloat16", F32, 4, 2, 128), ("float32", F32, 4, 2, 64)])
@pytest.mark.parametrize("h", [0, 130])
def test_a_key_with_a_score_of_minus_infinity_weighs_nothing(store, dtype, heads, g, dim, h):
    """The first drafted token's keys give every row -inf: as if no row saw it.  Rows that see only such keys are zeros."""
    requests = [(6, h), (3, 10)]
    c = Case(requests, heads, g, dim, 16, dtype, store, seed=11, spare_rows=0)
    x = c.q.view(-1, heads, dim)
    x[..., 3] = x[..., 3].abs() + 0.25
    c.cache[int(c.tables[0][h // 16]), 0, :, h % 16, 3] = -math.inf
    c.tree = ops.tree_bits([[-1, 0, 0, 1, 2, 2], [-1, 0, 1]])
    got = c.run()
    c.tree[:6] &= ~1
    assert torch.equal(got, c.run()) and bool(got.isfinite().all())
    assert bool((got[0] == 0).all()) == (h == 0)


@gpu
@pytest.mark.parametrize("n, h, claimed", [(100, 40, 100), (90, 500, 90), (100, 40, 101), (90, 500, 400)])
def test_rows_and_keys_beyond_what_was_said(n, h, claimed):
    """Counts on the device that the call's bounds do not cover: rows beyond the output's are not written, a request of more rows than
    `max_rows` is left alone, the others are what they were."""
    c = Case([(n, h), (2, 9)], 8, 2, 128, 16, BF16, seed=12, spare_rows=0)
    want, q = c.run(), c.q.to(DEV)
    for counts, max_rows, same in (([n, claimed], n, slice(0, n)), ([claimed, 2], n, slice(n, n + 2))):
        out = torch.full_like(q, 7.0)
        starts, _, histories, tables = c.device()
        ops.attention_quantized(q, c.cache, out, starts, torch.tensor(counts, dtype=torch.int32, device=DEV), histories, tables, c.heads, c.g, c.dim,
                                None, c.scale, max_rows, c.bounds()[1])
        assert torch.equal(out[same].double().cpu(), want[same])
        if claimed > max_rows:
            other = slice(n, n + 2) if counts[0] == n else slice(0, n)
            assert bool((out[other] == 7.0).all())
    out = torch.full_like(q, 7.0)
    ops.attention_quantized(q, c.cache, out, *c.device(), c.heads, c.g, c.dim, None, c.scale, n, max(h - 1, 20))      # fewer keys than there are
    assert torch.equal(out[n:].double().cpu(), want[n:])


@gpu
@pytest.mark.parametrize("heads, g, dim", [(8, 2, 128), (4, 2, 64)])
@pytest.mark.parametrize("n, h", [(5, 300), (200, 100), (300, 3000)])
@pytest.mark.parametrize("plane", [0, 1])
def test_rows_before_a_key_that_is_no_number_do_not_meet_it(heads, g, dim, n, h, plane):
    """A token in the middle of a portion with an infinity in one head's key or value: its own row and those behind it are NaN for
    the heads that read it, everything else is what it was."""
    c = Case([(n, h), (2, 9)], heads, g, dim, 16, BF16, seed=13, spare_rows=0)
    at = n // 2
    t = h + at
    page, place = int(c.tables[0][t // 16]), t % 16
    x = torch.randn(2, 1, g, dim, generator=torch.Generator().manual_seed(1)).to(DEV)
    slot = torch.tensor([page * 16 + place], dtype=torch.int32, device=DEV)
    ops.quantize_kv(x[0], x[1], slot, c.cache)
    want = c.run()
    x[plane, 0, 1, 3] = -math.inf
    ops.quantize_kv(x[0], x[1], slot, c.cache)
    got = c.run()
    hit = torch.zeros(c.rows, heads * dim, dtype=torch.bool)
    hit[at:n, heads // g * dim:2 * heads // g * dim] = True
    assert bool(got[hit].isnan().all())
    assert torch.equal(got[~hit], want[~hit])


@gpu
@pytest.mark.parametrize("rows", [1, 9, 200])
def test_pages_outside_of_the_cache_read_as_zeros(rows):
    c = Case([(rows, 500)], 8, 2, 128, 16, BF16, seed=8)
    c.tables[0, 3] = -1
    c.tables[0, 20] = -7
    c.check()
    c.tables[0, 3], c.tables[0, 20] = c.pages, 2 ** 31 - 1
    c.check()


@gpu
@pytest.mark.parametrize("size", [2.0 ** -45, 2.0 ** 45])
def test_keys_and_values_far_from_one(size):
    """Exponents near their ends in keys (with queries as far the other way) and in values."""
    c = Case([(2, 300), (1, 40)], 8, 2, 128, 16, BF16, seed=9)
    shift = round(math.log2(size))
    b = c.cache.exponents
    b[:, 0] = (b[:, 0].int() - shift).to(torch.uint8)
    b[:, 1] = (b[:, 1].int() + shift).to(torch.uint8)
    c.values[:, 0] *= 2.0 ** -shift
    c.values[:, 1] *= 2.0 ** shift
    c.q = (c.q.float() * 2.0 ** shift).to(BF16)
    c.check()


@gpu
def test_values_of_very_different_size():
    """The heaviest key has tiny values, keys of no weight have huge ones."""
    c = Case([(1, 700)], 4, 1, 128, 16, BF16, seed=10, spread=0.3)
    b = c.cache.exponents
    page, place = int(c.tables[0][200 // 16]), 200 % 16
    shift = torch.randint(-40, 1, (c.pages, 1, 16), generator=torch.Generator().manual_seed(1))
    b[:, 1] = (b[:, 1].int() + shift.to(DEV)).to(torch.uint8)
    c.values[:, 1] *= torch.exp2(shift.double())[..., None]
    c.q *= 8
    c.check()


@gpu
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_another_stream_and_a_recorded_call_over_changed_lengths(tree, dtype):
    requests = [(3, 200), (1, 900), (5, 31)]
    c = Case(requests, 8, 2, 128, 16, dtype, seed=11)
    if tree:
        c.tree = random_tree(requests, 11)
    want = c.run()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = c.run()
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want)
    # Recorded with these lengths as the most that there will be, replayed with shorter ones and with these again.
    q, out = c.q.to(DEV), torch.full_like(c.q.to(DEV), 7.0)
    start, count, history, tables = c.device()
    words = torch.from_numpy(c.tree).to(DEV) if tree else None

    def call():
        if tree:
            ops.attention_tree(q, c.cache, out, start, count, history, tables, words, 8, 2, 128, c.scale, *c.bounds())
        else:
            ops.attention_quantized(q, c.cache, out, start, count, history, tables, 8, 2, 128, None, c.scale, *c.bounds())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    shorter = Case(requests, 8, 2, 128, 16, dtype, seed=11)
    shorter.requests = [(2, 77), (1, 3), (5, 31)]
    shorter.tree = c.tree
    count.copy_(torch.tensor([2, 1, 5]))
    history.copy_(torch.tensor([77, 3, 31]))
    graph.replay()
    got = out.double().cpu()
    rows = [0, 1, 3, 4, 5, 6, 7, 8]
    call_want = torch.full_like(out, 7.0)
    o2, out = out, call_want
    call()
    assert torch.equal(got[rows], call_want.double().cpu()[rows])
    out = o2
    count.copy_(torch.tensor([3, 1, 5]))
    history.copy_(torch.tensor([200, 900, 31]))
    graph.replay()
    assert torch.equal(out[:c.rows].double().cpu(), want)


@gpu
def test_written_attended_and_read_back():
    """A request's tokens go in portion by portion; what attention gives after each is what attention over what reading back gives."""
    g, heads, dim, page, total = 2, 8, 128, 16, 300
    gen = torch.Generator().manual_seed(12)
    k, v = (torch.randn(total, g, dim, generator=gen) for _ in range(2))
    q = torch.randn(total, heads * dim, generator=gen).to(BF16)
    c = Case([(1, total - 1)], heads, g, dim, page, BF16, seed=12)
    slots = (c.tables[0].long()[torch.arange(total) // page] * page + torch.arange(total) % page).int()
    at = 0
    for n in (1, 7, 130, 1, 40, 121):
        ops.quantize_kv(k[at:at + n].to(DEV), v[at:at + n].to(DEV), slots[at:at + n].to(DEV), c.cache)
        ids = c.tables[0][:-(-(at + n) // page)].to(DEV)
        back = torch.empty(len(ids), 2, g, page, dim, device=DEV)
        ops.dequantize_pages(c.cache, ids, back)
        c.values = torch.zeros_like(c.values)
        c.values[ids.cpu().long()] = back.double().cpu()
        c.requests, c.starts, c.rows, c.q = [(n, at)], [0], n, q[at:at + n]
        c.check()
        at += n


# ---- as a step writes it, and in an engine ------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads, g, dim, page, rot_half, normed", [(8, 2, 128, 16, 64, True), (8, 8, 128, 32, 0, False), (6, 2, 64, 16, 32, True), (3, 1, 48, 8, 12, True),
                                                                   (5, 1, 128, 16, 48, True)])
def test_a_steps_rows_go_in_as_their_32_bit_ones_would(dtype, heads, g, dim, page, rot_half, normed):
    """Queries have the bits that they have over a cache of another type; keys and values are the 32-bit cache's, quantized."""
    gen = torch.Generator().manual_seed(dim)
    rows, n_pages = 37, 8
    qkv = torch.randn(rows, (heads + 2 * g) * dim, generator=gen).to(DEV)
    qkv[3, heads * dim + 5], qkv[4, -1] = math.inf, math.nan
    qw, kw = ((1 + 0.1 * torch.randn(dim, generator=gen)).to(DEV) for _ in range(2)) if normed else (None, None)
    angle = torch.rand(64, max(rot_half, 1), generator=gen).to(DEV) * 6
    cos, sin = (angle.cos().contiguous(), angle.sin().contiguous()) if rot_half else (None, None)
    positions = torch.randint(0, 64, (rows,), generator=gen).int().to(DEV)
    slots = torch.randperm(n_pages * page, generator=gen)[:rows].int().to(DEV)
    slots[7] = -1
    q32, q = torch.zeros(rows, heads * dim, device=DEV), torch.zeros(rows, heads * dim, dtype=dtype, device=DEV)
    plain, cache = torch.zeros(n_pages, 2, g, page, dim, device=DEV), ops.QuantizedPages.zeros(n_pages, g, page, dim, DEV)
    for out, store in ((q32, plain), (q, cache)):
        ops.head_norm_rope_kv(qkv, heads, g, dim, qw, kw, 1e-6, cos, sin, positions, slots, out, store)
    assert torch.equal(q, q32.to(dtype))
    values, b = quantized(plain.cpu().double().numpy())
    assert np.array_equal(cache.exponents.cpu().numpy(), b)
    want = np.where(b[..., None] == 255, np.nan, values * np.exp2(b[..., None] - 127.0))
    assert np.array_equal(decoded(cache.codes, cache.exponents), want, equal_nan=True)


@gpu
@pytest.mark.parametrize("requests", [[(1, 300), (1, 5), (1, 77)], [(200, 33), (1, 100), (3, 0)]])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_the_paged_kernels_entry_takes_eight_bits(requests, dtype):
    from llmx_b200 import ops_attn
    c = Case(requests, 8, 2, 128, 16, dtype, seed=14, spare_rows=0)
    step = ops_attn.attention_step(DEV, [(h, n) for n, h in requests], c.tables.clamp(min=0).numpy(), 8, 2, 128, None)

    class Same(Case):
        def run(self, window=None, out=None):
            out = torch.zeros_like(self.q.to(DEV))
            ops_attn.paged_attention(self.q.to(DEV), out, step, 0, 8, 2, 128, window, self.scale, cache=ops_attn.OneEntryCache(self.cache))
            return out.double().cpu()
    c.__class__ = Same
    c.check()


def _plain_logits(folder, ids, bf16):
    import helpers
    import plain_qwen3 as plain
    cfg, w = helpers._folder(folder)

    def in_eight_bits(x):
        values, b = quantized(np.asarray(x, dtype=np.float64))
        return (values * np.exp2(b[..., None] - 127.0)).astype(np.float32)
    return plain.forward(cfg, w, list(ids), act_round=plain.round_bf16 if bf16 else None, cache_round=in_eight_bits)


@gpu
@pytest.mark.parametrize("name", ["A", "B", "C", "D", "E"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("record", [False, True])
def test_an_engine_over_eight_bits(model_dirs, name, dtype, record):
    """Logits against the plain implementation that quantizes the same keys and values.  A key that falls on the other side of a
    rounding border moves a logit by 2e-3 of the scale where steps are bfloat16's (test_a_cache_type_of_its_own); a code's
    steps are 16 times as wide."""
    import helpers
    from configs import BF16_BUDGET, CONFIGS
    from llmx_b200.engine import Engine, EngineOptions
    d16, d32, page = model_dirs[name]
    folder = d32 if dtype == "float32" else d16
    vocab = CONFIGS[name][0]["vocab_size"]
    requests = {f"k{i}": helpers.random_ids(vocab, n, seed=90 + i) for i, n in enumerate([70, 9, 133, 33, 1])}
    steps = helpers.trace_tail_decoded(requests, 20) if record else helpers.trace_mixed(requests)
    engine = Engine.from_dir(folder, EngineOptions(dtype=dtype, kv_dtype="float8_e4m3", kv_tokens=helpers.tokens_needed(steps), page_size=page, max_requests=4,
                                                   record_after=3))
    assert engine.cache.groups[0].storage.dtype is torch.float8_e4m3fn
    got = helpers.run_trace(engine, steps, record=record)
    assert not record or engine.step_recordings
    engine.cache.check()
    for rid, ids in requests.items():
        ref = _plain_logits(folder, ids, dtype == "bfloat16")
        scale = float(np.abs(ref).max())
        worst = max(float(np.abs(got[(rid, p)] - ref[p]).max()) for p in range(len(ids)) if (rid, p) in got)
        assert worst <= (3.2e-2 + (BF16_BUDGET[name] if dtype == "bfloat16" else 0)) * scale, (rid, worst / scale)


@gpu
def test_generation_over_eight_bits(model_dirs):
    """The command's entry: greedy tokens with recorded decoding steps, the cache at an eighth of 32 bits and an exponent a row."""
    from llmx_b200.engine.generate import LLM
    from llmx_b200.sampling import SamplingParams
    folder = model_dirs["E"][1]
    prompts = [[3, 5, 7, 11] * 12, [9], [2, 4] * 50]
    outs = [LLM(folder, dtype="float32", kv_dtype=t, kv_tokens=1024).generate(prompts, SamplingParams(max_tokens=24, temp=0.0, top_k=0, top_p=1.0, ignore_eos=True))
            for t in ("float8_e4m3", "float8_e4m3", None)]
    assert [o.tokens for o in outs[0]] == [o.tokens for o in outs[1]]
    assert all(len(o.tokens) == 24 for o in outs[0])
    llm, wide = LLM(folder, dtype="float32", kv_dtype="f8", kv_tokens=1024), LLM(folder, dtype="float32", kv_tokens=1024)
    d = wide.engine.model.cache_entry_specs()[0].head_dim
    assert llm.engine.cache.storage_bytes() * 4 * d == wide.engine.cache.storage_bytes() * (d + 1)
